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
// nearest even, off by 2^-8 of the value at most; the sums of the product stay in 32 bits.
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
// The largest magnitude bits seen so far, two halves (bfloat16) or a word (float) at a time.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ inline uint32_t magnitude(uint32_t most, u32x4 v, __bf16) {
  u16x2 m = __builtin_bit_cast(u16x2, most);
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu));
  return __builtin_bit_cast(uint32_t, m);
}
__device__ inline uint32_t magnitude(uint32_t most, u32x4 v, float) {
#pragma unroll
  for (int i = 0; i < 4; ++i) most = max(most, v[i] & 0x7fffffffu);
  return most;
}
__device__ inline bool not_finite(uint32_t most, __bf16) { return (most & 0x7f80u) == 0x7f80u || (most >> 16) >= 0x7f80u; }
__device__ inline bool not_finite(uint32_t most, float) { return most >= 0x7f800000u; }
__device__ inline bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
template <typename F> __device__ inline F cleaned(F f) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (!finite((float)f[e])) f[e] = 0;
  return f;
}

// ---- rows in memory --------------------------------------------------------------------------
// Rows of one head: element d of row r at p + r * row + d, d < dim, dim <= row < 2^22 (checked by the
// host), so that a hundred rows are within reach of 32-bit byte offsets.  vec: 16-byte accesses are allowed
// (pointer and strides multiples of 16 bytes, dim a multiple of eight elements), decided by the host;
// kernels come in two forms, VEC for calls whose every array allows them.
//
// A run of rows is accessed through a buffer descriptor that ends behind its last row's last element: what lies outside
// reads as zero and is not written, so that odd lengths and head sizes cost no branch.
struct Rows {
  void *p;
  int64_t row, head;  // strides in elements
  int32_t dim, vec;
};

template <typename T> __device__ inline const T *head_of(const Rows &r, int head) {
  return (const T *)r.p + (int64_t)head * r.head;
}

typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ inline Buffer buffer_of(const void *p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, bytes, 0x00020000);
}
// Rows [first, first + count) of a head.  The descriptor's address has to be a multiple of four bytes: `lead` is
// how far the first row lies behind it.
struct Run {
  Buffer b;
  uint32_t lead;
};
//
// For reading, the end is moved up to a multiple of four bytes: element loads are made of whole words.  An allocation
// holds every word that it holds a byte of; what such a word has of others is masked.
template <typename T, bool READ = false> __device__ inline Run rows_buffer(const Rows &r, int head, int64_t first, int count) {
  // (the same for all lanes of a wave: said to the compiler, which would loop over the lanes' values otherwise)
  const uint64_t at = (uint64_t)(head_of<T>(r, head) + first * r.row);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)at), hi = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
  const uint32_t lead = lo & 3;
  uint32_t bytes = count > 0 ? ((uint32_t)(count - 1) * (uint32_t)r.row + (uint32_t)r.dim) * (uint32_t)sizeof(T) + lead : 0;
  if (READ) bytes = (bytes + 3) & ~3u;
  Run run;
  run.b = buffer_of((void *)(((uint64_t)hi << 32) | (lo & ~3u)), __builtin_amdgcn_readfirstlane(bytes));
  run.lead = lead;
  return run;
}
constexpr uint32_t kOutside = 0xfffffff0u;  // a byte offset behind every buffer's end

// Eight elements from d on of the row that starts `at` bytes into the buffer.  Words of a buffer may lie at any
// multiple of four bytes, so only two things keep rows of other sizes from being read like VEC's: bfloat16 at an odd
// place, for which a fifth word is read and the words are shifted, and what lies behind the row's end, which is
// masked.  settled() does both once the words are there (2739 rows x 12 x 77: forward 67 us with single loads, 39 us so).
template <typename T> __device__ inline void buffer_words8(Run u, uint32_t at, int d, int dim, bool vec, Frag<T> *f, uint32_t *fifth) {
  const uint32_t o = d < dim ? (vec ? at : u.lead + at) + d * (uint32_t)sizeof(T) : kOutside;
  if (sizeof(T) == 2) {
    const uint32_t w = o & ~3u;  // (outside stays outside)
    const u32x4 x = (u32x4)__builtin_amdgcn_raw_buffer_load_b128(u.b, vec ? o : w, 0, 0);
    __builtin_memcpy(f, &x, 16);
    if (!vec) *fifth = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(u.b, d < dim ? w + 16 : kOutside, 0, 0);
  } else {
    const u32x4 x = (u32x4)__builtin_amdgcn_raw_buffer_load_b128(u.b, o, 0, 0);
    const u32x4 y = (u32x4)__builtin_amdgcn_raw_buffer_load_b128(u.b, d < dim ? o + 16 : kOutside, 0, 0);
    __builtin_memcpy(f, &x, 16);
    __builtin_memcpy((char *)f + 16, &y, 16);
  }
}
// `left`: elements of the row from d on; `odd`: bytes that the first one lies behind its word's start.
__device__ inline bf16x8 settled(bf16x8 f, uint32_t fifth, uint32_t odd, int left) {
  u32x4 x = __builtin_bit_cast(u32x4, f);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t to = c < 3 ? x[c < 3 ? c + 1 : 3] : fifth;
    x[c] = __builtin_amdgcn_alignbyte(to, x[c], odd) & (left > 2 * c + 1 ? ~0u : left > 2 * c ? 0xffffu : 0u);
  }
  return __builtin_bit_cast(bf16x8, x);
}
__device__ inline f32x8 settled(f32x8 f, uint32_t, uint32_t, int left) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = e < left ? f[e] : 0.f;
  return f;
}
template <typename T> __device__ inline Frag<T> buffer_load8(Run u, uint32_t at, int d, int dim, bool vec) {
  Frag<T> f;
  uint32_t fifth = 0;
  buffer_words8<T>(u, at, d, dim, vec, &f, &fifth);
  return vec ? f : settled(f, fifth, (u.lead + at) & 3, dim - d);
}

// Whole pieces in one or two stores, bfloat16 at an odd place in three (its second to seventh elements are words); what
// ends the row element by element.
template <typename T> __device__ inline void buffer_store8(Run u, uint32_t at, int d, int dim, bool vec, Frag<T> f) {
  const uint32_t o = (vec ? at : u.lead + at) + d * (uint32_t)sizeof(T);
  const bool whole = vec ? d < dim : d + 8 <= dim && (o & 3) == 0;
  u32x4 w[sizeof(T) / 2];
  __builtin_memcpy(w, &f, sizeof(f));
#pragma unroll
  for (int c = 0; c < (int)sizeof(T) / 2; ++c) __builtin_amdgcn_raw_buffer_store_b128(w[c], u.b, whole ? o + 16 * c : kOutside, 0, 0);
  if (vec || whole || d >= dim) return;
  if constexpr (sizeof(T) == 2) {
    if (d + 8 <= dim) {
      typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));
      u32x3 x;
#pragma unroll
      for (int c = 0; c < 3; ++c) x[c] = __builtin_amdgcn_alignbyte(w[0][c + 1], w[0][c], 2);
      __builtin_amdgcn_raw_buffer_store_b16((short)w[0][0], u.b, o, 0, 0);
      __builtin_amdgcn_raw_buffer_store_b96(x, u.b, o + 2, 0, 0);
      __builtin_amdgcn_raw_buffer_store_b16((short)(w[0][3] >> 16), u.b, o + 14, 0, 0);
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const T x = f[e];
    const uint32_t to = d + e < dim ? o + e * (uint32_t)sizeof(T) : kOutside;
    if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, x), u.b, to, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), u.b, to, 0, 0);
  }
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
template <int D> __device__ inline bf16x8 col_frag(const __bf16 *t, int k0, int d0, int) { return col_frag<D>(t, k0, d0); }
template <int D> __device__ inline f32x8 col_frag(const float *t, int k0, int d0, int l = lane_id()) {
  const int d = d0 + pi_of(l & 31), row = k0 + ((l >> 5) << 3);
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
template <typename T, int D, int ROWS, int THREADS, bool VEC, bool FRESH = false> struct Staged {
  static constexpr int kPerRow = D / 8;
  static constexpr int kCount = ROWS * kPerRow / THREADS;
  static_assert(ROWS * kPerRow % THREADS == 0 && THREADS % kPerRow == 0, "whole pieces");
  static constexpr int kStep = THREADS / kPerRow;  // rows from one of a thread's pieces to its next
  static_assert(kStep % 2 == 0, "all of a thread's rows start at odd places or none");
  static constexpr bool kFifth = !VEC && sizeof(T) == 2;
  Frag<T> f[kCount];
  uint32_t fifth[kFifth ? kCount : 1], odd;
  int left;
  // rows first + r, or with `back` first - r, for r in [0, count) are read, the others become zeros
  __device__ inline void load(const Rows &rows, int head, int64_t first, bool back, int count) {
    const int tid = threadIdx.x % THREADS, r0 = tid / kPerRow, d = (tid % kPerRow) * 8;
    const Run b = rows_buffer<T, !VEC>(rows, head, back ? first - (count - 1) : first, count);
    const int row = (int)rows.row * (int)sizeof(T);
    // (backwards, rows from `count` on lie before the buffer: offsets below zero, which are outside too)
    int at = back ? (count - 1 - r0) * row : r0 * row;
    const int step = (back ? -kStep : kStep) * row;
    if (FRESH) asm volatile("" : "+v"(at));  // (the pieces' offsets are worked out anew each time: cheaper than registers)
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int dim = VEC || r0 + i * kStep < count ? rows.dim : 0;
      buffer_words8<T>(b, at + i * step, d, dim, VEC, &f[i], &fifth[kFifth ? i : 0]);
    }
    odd = (b.lead + at) & 3;
    left = rows.dim - d;
  }
  // the words into elements, before they are looked at or stored
  __device__ inline void settle() {
    if (VEC) return;
#pragma unroll
    for (int i = 0; i < kCount; ++i) f[i] = settled(f[i], fifth[kFifth ? i : 0], odd, left);
  }
  __device__ inline void store(T *t) const {
    const int tid = threadIdx.x % THREADS, r0 = tid / kPerRow, d = (tid % kPerRow) * 8;
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int r = r0 + i * kStep;
      const u32x4 *w = (const u32x4 *)&f[i];
#pragma unroll
      for (int c = 0; c < (int)sizeof(T) / 2; ++c)
        *(u32x4 *)((char *)t + tile_at<T, D>(r, d + c * (16 / (int)sizeof(T)))) = w[c];
    }
  }
  __device__ inline void clean() {  // zeros in place of what is not finite
#pragma unroll
    for (int i = 0; i < kCount; ++i) f[i] = cleaned(f[i]);
  }
  __device__ inline bool dirty() const {  // whether a value is not finite
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kCount; ++i)
#pragma unroll
      for (int c = 0; c < (int)sizeof(T) / 2; ++c) most = magnitude(most, ((const u32x4 *)&f[i])[c], T());
    return not_finite(most, T());
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

// How many offsets are <= row, found by all lanes of the wave together, 64 places a step.
__device__ inline int count_le(const Series &s, int64_t row) {
  if (!s.offsets) return 1;
  int lo = 0, hi = s.n_series + 1;
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

// Sixty-four consecutive offsets, one a lane (-1 before the first, past every row behind the last): the series of
// near rows are found in them without further loads.
struct Offsets {
  int base;  // of lane 0
  int o;
};
__device__ inline Offsets offsets_from(const Series &s, int base) {
  Offsets w;
  w.base = base;
  const int i = base + lane_id();
  if (!s.offsets) {
    w.o = i < 0 ? -1 : i == 0 ? 0 : i == 1 ? s.n : kNoSeries;
  } else {
    const int64_t x = s.offsets[i < 0 ? 0 : i > s.n_series ? s.n_series : i];
    w.o = i < 0 ? -1 : i > s.n_series ? kNoSeries : x < 0 ? 0 : x > s.n ? s.n : (int)x;
  }
  return w;
}
// The window of offsets around `row`, most of it behind (back: before) it.
__device__ inline Offsets offsets_at(const Series &s, int row, bool back) {
  const int c = count_le(s, row);
  return offsets_from(s, back ? c - 62 : c - 1);
}
// The series of `row` (the same for all lanes).  A stretch of rows that belong to none has index -1.
__device__ inline Span span_of(const Series &s, Offsets &w, int row, bool back) {
  uint64_t past = __ballot(w.o > row);
  if (past == 0 || (past & 1)) {  // not in the window
    w = offsets_at(s, row, back);
    past = __ballot(w.o > row);
  }
  // (offsets that do not ascend may leave nothing here: the row then stands alone)
  const int l = past == 0 || (past & 1) ? -1 : __builtin_ctzll(past);
  Span sp = {row, row + 1, -1};
  if (l < 0) return sp;
  const int a = __builtin_amdgcn_readlane(w.o, l - 1), b = __builtin_amdgcn_readlane(w.o, l);
  sp.start = a < 0 ? 0 : a;
  sp.end = b > s.n ? s.n : b;
  const int i = w.base + l - 1;
  sp.index = i < 0 || i >= s.n_series ? -1 : i;
  return sp;
}
// The series of each lane's own row, one of [first, last]; the window is the one of `first`.
__device__ inline Span lane_span(const Series &s, const Offsets &w, int first, int last, int row) {
  const int l0 = __popcll(__ballot(w.o <= first)), l1 = __popcll(__ballot(w.o <= last));
  int a, b, i;
  if (l1 < 64) {
    int c = l0;
    for (int l = l0; l < l1; ++l) c += __builtin_amdgcn_readlane(w.o, l) <= row;
    a = __shfl(w.o, c - 1);
    b = __shfl(w.o, c);
    i = w.base + c - 1;
  } else {  // more series start among these rows than the window holds: each lane looks for its own
    int lo = w.base < 0 ? 0 : w.base, hi = s.n_series + 1;
    while (lo < hi) {
      const int mid = lo + ((hi - lo) >> 1);
      if (s.offsets[mid] <= row) lo = mid + 1; else hi = mid;
    }
    i = lo - 1;
    const int64_t x = s.offsets[i < 0 ? 0 : i], y = s.offsets[i >= s.n_series ? s.n_series : i + 1];
    a = (int)(x < 0 ? 0 : x > s.n ? s.n : x);
    b = (int)(y < 0 ? 0 : y > s.n ? s.n : y);
  }
  Span sp = {kNoSeries, row + 1, -1};
  if (i < 0 || i >= s.n_series || a > row || b <= row) return sp;
  sp.start = a;
  sp.end = b;
  sp.index = i;
  return sp;
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
// Without offsets there is one series, also where n_series was left zero; numbers of series are compared with 32-bit
// arithmetic beside that of rows.
inline bool series_ok(const int64_t *offsets, int32_t n_series) {
  return n_series >= 0 && n_series < (offsets ? kNoSeries : 2);
}
#define TMP_SERIES(what, a)                                                                                     \
  TMP_REQUIRE(series_ok((a)->offsets, (a)->n_series), TMP_EINVAL,                                               \
              "%s: bad series: their number must be in [0, 2^31 - 65536), at most 1 without offsets", what)
// Rows of `n`, dim elements each; false: strides that the kernels do not take.
inline bool rows_of(const tmp_rows &r, int64_t n, int dim, int bytes, Rows *o) {
  const int64_t per = 16 / bytes;
  o->p = r.p; o->row = n > 1 ? r.row_stride : (dim + 7) / 8 * 8; o->head = r.head_stride; o->dim = dim;
  o->vec = ((uintptr_t)r.p & 15) == 0 && o->row % per == 0 && r.head_stride % per == 0 && dim % 8 == 0;
  return o->row >= dim && o->row < (1 << 22) && (uintptr_t)r.p % bytes == 0;
}
#define TMP_ROWS(what, ref, n, dim, bytes, to)                                                                 \
  TMP_REQUIRE(rows_of(ref, n, dim, bytes, to), TMP_EUNSUPPORTED,                                               \
              "%s: the row stride of " #ref " must be at least its head size and below 2^22 elements, its pointer aligned", what)

// A launch has fewer than 2^32 threads, so that one of blocks of 256 has fewer blocks than this (rounded down to eight,
// for grids that are a multiple of it).
constexpr int64_t kMostBlocks = (1 << 24) - 8;

// fn<T, D, VEC>(...) for a type, a padded head size and an access width.
#define TMP_BY_DIM(fn, T, d, VEC, ...)              \
  do {                                              \
    if ((d) == 32) fn<T, 32, VEC>(__VA_ARGS__);     \
    else if ((d) == 64) fn<T, 64, VEC>(__VA_ARGS__); \
    else fn<T, 128, VEC>(__VA_ARGS__);              \
  } while (0)
#define TMP_BY_FORM(fn, type, d, vec, ...)                             \
  do {                                                                 \
    if ((type) == TMP_F32) {                                           \
      if (vec) TMP_BY_DIM(fn, float, d, true, __VA_ARGS__);            \
      else TMP_BY_DIM(fn, float, d, false, __VA_ARGS__);               \
    } else {                                                           \
      if (vec) TMP_BY_DIM(fn, __bf16, d, true, __VA_ARGS__);           \
      else TMP_BY_DIM(fn, __bf16, d, false, __VA_ARGS__);              \
    }                                                                  \
  } while (0)

inline int padded_dim(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

}  // namespace tmp
