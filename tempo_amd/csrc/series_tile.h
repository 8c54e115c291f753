// Shared pieces of the attention kernels (window_attention.hip, decay_attention.hip): where a row's
// series starts, row tiles in LDS, and 32x32 matrix-core products of them.
//
// Fragments.  A wave multiplies with v_mfma_f32_32x32x16_bf16 (or eight v_mfma_f32_32x32x2_f32 for
// float): lane l holds, of either operand, row l % 32 and the eight k = 8 * (l / 32) + e of a step of
// sixteen.  The result's column is l % 32, and its register r is row 8 * (r / 4) + 4 * (l / 32) + r % 4.
// Every left operand is read with rows and columns passed through pi(), which swaps bits 2 and 3 of
// the row: register r then stands for row 16 * (r / 8) + 8 * (l / 32) + r % 8, so that eight
// consecutive registers are just what the next product's operand holds -- scores go into the product
// with the values, and a state into the product with the queries, without leaving the registers --
// and a lane's results are runs of eight consecutive elements of a row.
//
// Tiles.  Row-major in LDS, 16-byte chunks XORed with a function of the row (swz) such that sixteen
// lanes reading one chunk column of sixteen rows, and thirty-two lanes reading 4 rows x 64 bytes
// (ds_read_b64_tr_b16), touch all 64 banks once.
#pragma once

#include "common.h"

namespace tmp {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

template <typename T> struct FragOf;
template <> struct FragOf<__bf16> { typedef bf16x8 type; };
template <> struct FragOf<float> { typedef f32x8 type; };
template <typename T> using Frag = typename FragOf<T>::type;

__device__ inline float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline float log2_hw(float x) { return __builtin_amdgcn_logf(x); }
__device__ inline int lane_id() { return threadIdx.x & 63; }
__device__ inline int pi_of(int i) { return (i & 0x13) | ((i & 4) << 1) | ((i & 8) >> 1); }

__device__ inline f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

__device__ inline f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

// Registers 8 * b .. 8 * b + 7 of a result as the operand of a product's step b.  To bf16: rounded to
// nearest even, half a step of 2^-8 relative at most; the sums of the product stay in 32 bits.
template <typename T> __device__ inline Frag<T> operand(const f32x16 &c, int b);
template <> __device__ inline bf16x8 operand<__bf16>(const f32x16 &c, int b) {
  bf16x8 f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    f32x2 v = {c[8 * b + e], c[8 * b + e + 1]};
    bf16x2 w = __builtin_convertvector(v, bf16x2);
    f[e] = w[0];
    f[e + 1] = w[1];
  }
  return f;
}
template <> __device__ inline f32x8 operand<float>(const f32x16 &c, int b) {
  f32x8 f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = c[8 * b + e];
  return f;
}

// ---- values that are not finite -------------------------------------------------------------
// A masked position must not reach a result, and 0 * NaN would.  Tiles are looked at as they are
// staged; a tile that holds such a value (rare) has its operands cleaned and the visible ones added.
__device__ inline uint32_t not_finite(u32x4 v, __bf16) {  // nonzero if a half has all exponent bits set
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= ((v[i] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
  return bad;
}
__device__ inline uint32_t not_finite(u32x4 v, float) {
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= ((v[i] & 0x7f800000u) + 0x00800000u) & 0x80000000u;
  return bad;
}
__device__ inline bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
template <typename F> __device__ inline F cleaned(F f) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (!finite((float)f[e])) f[e] = 0;
  return f;
}

// ---- rows in memory --------------------------------------------------------------------------
// Rows of one head: element d of row r at p + r * stride + d, d < dim.  vec: 16-byte loads are allowed
// (pointer and strides multiples of 16 bytes, dim a multiple of eight elements), decided by the host.
struct Rows {
  void *p;
  int64_t row, head;  // strides in elements
  int32_t dim, vec;
};

template <typename T> __device__ inline const T *head_of(const Rows &r, int head) {
  return (const T *)r.p + (int64_t)head * r.head;
}

// Eight elements from d on of the row at `p`, zeros beyond dim.
__device__ inline bf16x8 load8(const __bf16 *p, int d, int dim, bool vec) {
  bf16x8 f;
  if (vec && d < dim) return *(const bf16x8 *)(p + d);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = d + e < dim ? p[d + e] : (__bf16)0.f;
  return f;
}
__device__ inline f32x8 load8(const float *p, int d, int dim, bool vec) {
  f32x8 f;
  if (vec && d < dim) {
    const f32x4 a = *(const f32x4 *)(p + d), b = *(const f32x4 *)(p + d + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) { f[e] = a[e]; f[e + 4] = b[e]; }
    return f;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = d + e < dim ? p[d + e] : 0.f;
  return f;
}
template <typename F> __device__ inline F zero_frag() {
  F f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = 0;
  return f;
}
__device__ inline void store8(__bf16 *p, int d, int dim, bool vec, bf16x8 f) {
  if (vec && d < dim) { *(bf16x8 *)(p + d) = f; return; }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (d + e < dim) p[d + e] = f[e];
}
__device__ inline void store8(float *p, int d, int dim, bool vec, f32x8 f) {
  if (vec && d < dim) {
    f32x4 a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) { a[e] = f[e]; b[e] = f[e + 4]; }
    *(f32x4 *)(p + d) = a;
    *(f32x4 *)(p + d + 4) = b;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (d + e < dim) p[d + e] = f[e];
}

// ---- tiles in LDS ----------------------------------------------------------------------------
// `D` columns (a power of two from 32 to 128) of T.
template <typename T, int D> __device__ inline int swz(int row) {
  constexpr int bytes = D * (int)sizeof(T);
  if constexpr (sizeof(T) == 2) {
    if constexpr (bytes == 256) return ((row & 3) << 2) | ((row >> 2) & 3);
    else if constexpr (bytes == 128) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    else return (row >> 2) & 3;
  } else {
    if constexpr (bytes == 128) return (row >> 1) & 7;
    else return row & 15;
  }
}
// Byte offset of element `d` (a multiple of the 16-byte chunk, or any for single elements) of `row`.
template <typename T, int D> __device__ inline int tile_at(int row, int d) {
  constexpr int per = 16 / (int)sizeof(T);
  const int chunk = d / per, in = d % per;
  return row * (D * (int)sizeof(T)) + ((chunk ^ swz<T, D>(row)) << 4) + in * (int)sizeof(T);
}

template <int D> __device__ inline bf16x8 row_frag(const __bf16 *t, int row, int d) {
  return *(const bf16x8 *)((const char *)t + tile_at<__bf16, D>(row, d));
}
template <int D> __device__ inline f32x8 row_frag(const float *t, int row, int d) {
  const f32x4 a = *(const f32x4 *)((const char *)t + tile_at<float, D>(row, d));
  const f32x4 b = *(const f32x4 *)((const char *)t + tile_at<float, D>(row, d + 4));
  f32x8 f;
#pragma unroll
  for (int e = 0; e < 4; ++e) { f[e] = a[e]; f[e + 4] = b[e]; }
  return f;
}
// Left operand of a product over rows: lane l holds column d0 + pi(l % 32) of rows k0 + 8 * (l / 32) + e.
template <int D> __device__ inline bf16x8 col_frag(const __bf16 *t, int k0, int d0) {
  typedef __attribute__((address_space(3))) s16x4 *lds;
  const int l = lane_id(), i = l & 15;
  // the four 4-column pieces of a group of sixteen lanes, passed through pi: 0, 2, 1, 3 of this
  // half; lanes 16..31 hold columns 16..31
  const int c = i & 3;
  const int piece = ((c & 1) << 1) | (c >> 1);
  const int row = k0 + ((l >> 5) << 3) + (i >> 2);
  const int d = d0 + (((l >> 4) & 1) << 4) + piece * 4;
  const char *p = (const char *)t;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(p + tile_at<__bf16, D>(row, d)));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(p + tile_at<__bf16, D>(row + 4, d)));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  s16x8 f;
#pragma unroll
  for (int e = 0; e < 4; ++e) { f[e] = lo[e]; f[e + 4] = hi[e]; }
  return __builtin_bit_cast(bf16x8, f);
}
template <int D> __device__ inline f32x8 col_frag(const float *t, int k0, int d0) {
  const int l = lane_id(), d = d0 + pi_of(l & 31), row = k0 + ((l >> 5) << 3);
  f32x8 f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = *(const float *)((const char *)t + tile_at<float, D>(row + e, d));
  return f;
}
template <typename T, int D> __device__ inline float tile_elem(const T *t, int row, int d) {
  return (float)*(const T *)((const char *)t + tile_at<T, D>(row, d));
}

// A tile on its way from memory to LDS, by THREADS consecutive threads of the block: loads are issued by load(), waited for and written by store(),
// so that a tile travels while the one before it is worked on.
template <typename T, int D, int ROWS, int THREADS> struct Staged {
  static constexpr int kPerRow = D / 8;
  static constexpr int kCount = (ROWS * kPerRow + THREADS - 1) / THREADS;
  Frag<T> f[kCount];
  // rows first + step * r for r in [0, count) are read, the others become zeros
  __device__ inline void load(const T *p, int64_t row_stride, int dim, bool vec, int64_t first, int step, int count) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int at = threadIdx.x % THREADS + i * THREADS, r = at / kPerRow, d = (at % kPerRow) * 8;
      f[i] = r < count && d < dim ? load8(p + (first + (int64_t)step * r) * row_stride, d, dim, vec) : zero_frag<Frag<T>>();
    }
  }
  __device__ inline uint32_t store(T *t) const {  // whether it holds a value that is not finite
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int at = threadIdx.x % THREADS + i * THREADS, r = at / kPerRow, d = (at % kPerRow) * 8;
      if (ROWS * kPerRow % THREADS && r >= ROWS) continue;
      const u32x4 *w = (const u32x4 *)&f[i];
#pragma unroll
      for (int c = 0; c < (int)sizeof(T) / 2; ++c) {
        bad |= not_finite(w[c], T());
        *(u32x4 *)((char *)t + tile_at<T, D>(r, d + c * (16 / (int)sizeof(T)))) = w[c];
      }
    }
    return bad;
  }
};

// ---- series ----------------------------------------------------------------------------------
// offsets[0..n_series] are the first rows of the series, ascending, the last one the end of all; rows
// outside belong to none.  A null pointer is one series of all rows.  Values are only ever compared
// with rows of the table, so that wrong ones give wrong series and no access out of range.
struct Series {
  const int64_t *offsets;
  int32_t n_series;
  int32_t n;  // rows
};
struct Span {
  int start, end;  // rows [start, end) of the series; start = kNoSeries: the row belongs to none
  int index;
};
constexpr int kNoSeries = 0x7fff0000;  // beyond every row: tables have fewer than 2^31 - 65536

__device__ inline Span span_at(const Series &s, int count, int row) {  // count = offsets that are <= row
  Span sp;
  if (!s.offsets) { sp.start = 0; sp.end = s.n; sp.index = 0; return sp; }
  if (count < 1 || count > s.n_series) { sp.start = kNoSeries; sp.end = row + 1; sp.index = -1; return sp; }
  const int64_t a = s.offsets[count - 1], b = s.offsets[count];
  sp.start = a < 0 ? 0 : a > row ? row : (int)a;
  sp.end = b > s.n ? s.n : b <= row ? row + 1 : (int)b;
  sp.index = count - 1;
  return sp;
}
// How many offsets are <= row, found by all lanes of the wave together, 64 places a step; the answer is
// known to be in [lo, hi].
__device__ inline int count_le(const Series &s, int64_t row, int lo, int hi) {
  if (!s.offsets) return 1;
  while (lo < hi) {
    const int step = (hi - lo + 63) / 64;
    const int64_t at = (int64_t)lo + (int64_t)(lane_id() + 1) * step - 1;
    const bool le = at < hi && s.offsets[at] <= row;
    const int c = __popcll(__ballot(le));
    lo += c * step;
    const int top = lo + step - 1;
    hi = top < hi ? top : hi;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}
// The same for the lane's own row, between the counts of the tile's first and last rows.
__device__ inline int count_le_lane(const Series &s, int64_t row, int lo, int hi) {
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);
    if (s.offsets[mid] <= row) lo = mid + 1; else hi = mid;
  }
  return lo;
}

__device__ inline float other_half(float x) { return __shfl_xor(x, 32); }
__device__ inline int wave_max(int x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) { const int y = __shfl_xor(x, o); x = y > x ? y : x; }
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ inline int wave_min(int x) { return -wave_max(-x); }

// Blocks go to the eight dies in turn; consecutive work items share rows, so each die gets a run of them.
__device__ inline int item_of_block(int total) {
  const int per = (total + 7) / 8;
  const int item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  return (int)(blockIdx.x >> 3) < per && item < total ? item : -1;
}
inline int grid_of_items(int64_t total) { return (int)((total + 7) / 8 * 8); }

// ---- host side -------------------------------------------------------------------------------
inline Rows rows_of(const tmp_rows &r, int dim, int bytes) {
  Rows o;
  o.p = r.p; o.row = r.row_stride; o.head = r.head_stride; o.dim = dim;
  const int64_t per = 16 / bytes;
  o.vec = ((uintptr_t)r.p & 15) == 0 && r.row_stride % per == 0 && r.head_stride % per == 0 && dim % 8 == 0;
  return o;
}
inline int padded_dim(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

}  // namespace tmp
