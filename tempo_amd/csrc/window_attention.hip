// Attention over a sliding window of each series, with a few first rows that stay visible.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i),  lse_i = log sum_j exp(scale q_i.k_j)
//   j of i's series with j <= i and (j > i - window or j < start + sinks)
//
// and backward, with dP_ij = do_i.v_j and dS_ij = p_ij (dP_ij - do_i.o_i):
//   dq_i = scale sum_j dS_ij k_j    dk_j = scale sum_i dS_ij q_i    dv_j = sum_i p_ij do_i
//
// One skeleton serves all three kernels: a wave owns 32 rows, one per column of the matrix cores'
// result (its operands of them stay in registers), and the block's four waves stream the other side's
// rows through LDS in tiles of 64.  A row's scores then lie in two lanes, so the running maximum and
// sum of the softmax are lane-local but for one exchange, and scores turn into operands in place.
#include <string.h>

#include "row_limits.h"
#include "series_tile.h"

namespace tmp {

constexpr int WA_OWN = 128;    // rows that a block owns, 32 to each wave
constexpr int WA_TILE = 64;    // rows of a streamed tile
constexpr int WA_THREADS = 256;
constexpr int WA_SECTION = WA_OWN;  // query rows whose share of the sinks' gradients one block adds up

// bfloat16: dS enters dq and dk as the sum of two numbers at every window, since its own rounding would come on top of those
// of the result and of do.o (of the rounded out).  Error against 64 bits where rounding the result alone is 1.66e-3, two
// numbers | one: dq at window 1000, head size 64 1.82e-3 | 2.48e-3; dk 1.80e-3 | 2.44e-3, at window 70 1.75e-3 | 2.41e-3, at
// 11 2.00e-3 | 2.60e-3.  32768 x 16 x 64, window 1000: dq 300 | 250 us, dk and dv 406 | 350 us.  The weights P enter out and
// dv as one number (out 2.1e-3, dv 2.3e-3): a sum of rounded positive terms, whose second product would cost as much again.

struct WindowParams {
  Series s;
  Rows q, k, v, out, dout, dq, dk, dv;
  float *lse;    // [n][heads]
  float *delta;  // [n][heads], do_i.o_i
  float *sink_part;  // [sections][2][kv_heads][sinks][dk + dv]
  int32_t heads, kv_heads, window, sinks;
  float scale;
};

__device__ inline int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
__device__ inline int min_of(int a, int b) { return a < b ? a : b; }
__device__ inline int max_of(int a, int b) { return a > b ? a : b; }

// Which rows of a streamed tile a lane's own row sees (or is seen by): the run [lo, hi], and [slo, shi] of the rows
// that stay visible.
struct Seen {
  int lo, hi, slo, shi;
  __device__ inline bool operator()(int x) const { return ((x >= lo) & (x <= hi)) | ((x >= slo) & (x <= shi)); }
};
// Weights (or scores) x of a part whose first row is `at` (of the tile, for the lane's half): `off` where not seen.
template <bool SINKS> __device__ inline void mask_part(f32x16 &s, const Seen &seen, int at, float off) {
  const int lo = seen.lo - at, n = max_of(seen.hi - seen.lo + 1, 0), slo = seen.slo - at, sn = max_of(seen.shi - seen.slo + 1, 0);
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    const int r = 16 * (x >> 3) + (x & 7);
    bool on = (uint32_t)(r - lo) < (uint32_t)n;
    if (SINKS) on |= (uint32_t)(r - slo) < (uint32_t)sn;
    s[x] = on ? s[x] : off;
  }
}


// What a wave knows of its 32 own rows when they are query rows.
struct QueryRows {
  int i, start;               // the lane's row and where its series starts (i + 1: none)
  int lo, first_start;        // of the block: first row in any window, start of its first row's series
  int wmin, wmax, wlo, wstart;  // of the wave: first and last row, first row in any window, last start
  bool all;                   // every row of the wave lies in a series
  // Whether the wave may see any of `rows` rows from j0 on.
  __device__ inline bool any(const WindowParams &p, int j0, int rows) const {
    return j0 <= wmax && (j0 + rows > wlo || j0 < wstart + p.sinks);
  }
};

__device__ inline QueryRows query_rows(const WindowParams &p, int t0) {
  QueryRows r;
  const int t1 = t0 + WA_OWN < p.s.n ? t0 + WA_OWN : p.s.n;
  Offsets w = offsets_at(p.s, t0, false);
  const Span first = span_of(p.s, w, t0, false);
  r.i = t0 + wave_id() * 32 + (lane_id() & 31);
  r.first_start = first.index < 0 ? t0 : first.start;
  const int back = t0 - p.window + 1;
  r.lo = back > r.first_start ? back : r.first_start;
  const Span mine = lane_span(p.s, w, t0, t1 - 1, r.i);
  const bool in = r.i < t1 && mine.start <= r.i;
  r.start = in ? mine.start : r.i + 1;
  r.wmin = t0 + wave_id() * 32;
  r.wmax = r.wmin + 31;
  const int lo = r.i - p.window + 1 > r.start ? r.i - p.window + 1 : r.start;
  r.wlo = wave_min(lo);
  r.wstart = wave_max(r.start);
  r.all = __all(in);
  return r;
}

// The tiles of rows that query rows look at: the first series' sinks that lie before every window
// (part 0), then all rows from the first window on (part 1).
struct KeyTiles {
  int a0, a1, b0, b1, na, count;
  __device__ inline KeyTiles(const WindowParams &p, const QueryRows &r, int t0) {
    a0 = r.first_start;
    a1 = a0 + p.sinks < r.lo ? a0 + p.sinks : r.lo;
    if (a1 < a0) a1 = a0;
    b0 = r.lo;
    b1 = t0 + WA_OWN < p.s.n ? t0 + WA_OWN : p.s.n;
    na = (a1 - a0 + WA_TILE - 1) / WA_TILE;
    count = na + (b1 - b0 + WA_TILE - 1) / WA_TILE;
  }
  __device__ inline int first(int t) const { return t < na ? a0 + t * WA_TILE : b0 + (t - na) * WA_TILE; }
  __device__ inline int end(int t) const { return t < na ? a1 : b1; }
  __device__ inline int rows(int t) const {
    const int left = end(t) - first(t);
    return left < WA_TILE ? left : WA_TILE;
  }
};

// A masked row's weight of zero does not keep a value that is not finite out of a product.  A tile that holds such
// values (rare) is cleaned before it is multiplied, and what the lane's own row sees of them is added here first.
// By element: as they are, for products whose weights are positive.
template <typename T, int D, int ROWS = WA_TILE, int NT> __device__ inline void add_not_finite(f32x16 (&acc)[NT], const T *tile, Seen seen) {
  const int h8 = (lane_id() >> 5) * 8;
#pragma unroll 1
  for (int j = 0; j < ROWS; ++j) {
    const bool on = seen(j);
    int row = j;
    asm volatile("" : "+v"(row));  // keeps the addresses below out of the registers of the main path
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = tile_elem<T, D>(tile, row, t * 32 + 16 * (r >> 3) + h8 + (r & 7));
        acc[t][r] += on && !finite(x) ? x : 0.f;
        if ((r & 3) == 3) __builtin_amdgcn_sched_barrier(0);
      }
  }
}
// By row: NaN for every element, where the weight itself depends on such a value.
template <typename T, int D, int ROWS = WA_TILE, int NT> __device__ inline void mark_not_finite(f32x16 (&acc)[NT], const T *tile, Seen seen) {
  bool bad = false;
#pragma unroll 1
  for (int j = 0; j < ROWS; ++j) {
    bool any = false;
    for (int d = lane_id(); d < D; d += 64) any |= !finite(tile_elem<T, D>(tile, j, d));
    bad |= __any(any) & seen(j);
  }
  const float x = bad ? __uint_as_float(0x7fc00000u) : 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[t][r] += x;
}

// acc += (32 rows of the tile)^T w, for the lane's column of weights.
template <typename T, int D, int NT>
__device__ inline void add_rows(f32x16 (&acc)[NT], const T *tile, int row0, const f32x16 &w) {
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const Frag<T> wf = operand<T>(w, b);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const Frag<T> f = col_frag<D>(tile, row0 + 16 * b, t * 32);
      acc[t] = mma(f, wf, acc[t]);
    }
  }
}

// The same with the lane's number given, for places that are to be worked out anew.
template <int D, int NT>
__device__ inline void add_rows_at(f32x16 (&acc)[NT], const float *tile, int row0, const f32x16 &w, int l) {
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const f32x8 wf = operand<float>(w, b);
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = mma(col_frag<D>(tile, row0 + 16 * b, t * 32, l), wf, acc[t]);
  }
}

// How the instructions up to here are to follow each other: LDS reads for AHEAD matrix instructions first, then one
// matrix instruction, the reads (READS) of a later one and `valu` vector instructions in turn, so that neither the reads
// nor the vector unit wait for the matrix core or it for them.
template <int COUNT, int READS, int AHEAD, int VALU> __device__ inline void side_by_side() {
  __builtin_amdgcn_sched_group_barrier(0x100, READS * AHEAD, 0);
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (i + AHEAD < COUNT) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    if (VALU) __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
  }
}
// Keeps the computation of a value from being moved behind this place.
__device__ inline void hold(f32x16 &x) { asm volatile("" : "+v"(x)); }

// What rounding a part's weights to the operand's type leaves of them.
template <typename T> __device__ inline f32x16 left_over(f32x16 w) {
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const Frag<T> f = operand<T>(w, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[8 * b + e] -= (float)f[e];
  }
  return w;
}

// The lane's own row, row `r` of the buffer.  Rows of no series (in = false) are zeros.
template <typename T, int D, bool VEC>
__device__ inline void load_own(Frag<T> (&f)[D / 16], const Rows &rows, Run buf, int r, bool in) {
  const uint32_t at = in ? (uint32_t)r * (uint32_t)rows.row * (uint32_t)sizeof(T) : kOutside;
  const int h8 = 8 * (lane_id() >> 5), dim = in ? rows.dim : 0;
#pragma unroll
  for (int b = 0; b < D / 16; ++b) f[b] = buffer_load8<T>(buf, at, 16 * b + h8, dim, VEC);
}
template <typename T, int D, bool VEC, int NT>
__device__ inline void store_own(const f32x16 (&acc)[NT], float by, const Rows &rows, Run buf, int r) {
  const uint32_t at = (uint32_t)r * (uint32_t)rows.row * (uint32_t)sizeof(T);
  const int h8 = 8 * (lane_id() >> 5);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    f32x16 c = acc[t];
#pragma unroll
    for (int x = 0; x < 16; ++x) c[x] *= by;
#pragma unroll
    for (int b = 0; b < 2; ++b) buffer_store8<T>(buf, at, t * 32 + 16 * b + h8, rows.dim, VEC, operand<T>(c, b));
  }
}

// An element of a part costs 4 D operations and some ten vector instructions (scale, maximum, exponential, sum, rounding),
// which take as long as the products at D = 64 and half as long at 128.  131072 x 16 x 128, window 600: 1.09 ms, 583
// TFLOP/s of visible pairs; 32768 x 16 x 64, window 1000: 216 us, 537 TFLOP/s (library products reach 1134).  At 64 vector
// issue bounds it (0.64 of the cycles); at 128 nothing is full (matrix cores 0.31, vector issue 0.42, LDS 0.26): the chain
// product, maximum, exponential, product of 32 rows is waited for by two waves a SIMD.  Waves a SIMD: as many as fit the
// registers but for a few values (spilled: bf16 of 128 two, twelve for rows of odd sizes; float of 128 25 to 28).
template <typename T, int D, bool VEC>
__global__ __launch_bounds__(WA_THREADS, D * sizeof(T) == 128 ? 3 : 2) void window_forward_kernel(WindowParams p, int tiles) {
  // float: matrix instructions are a sixteenth as fast, and parts that a wave does not see are left out one by one
  constexpr int PARTS = sizeof(T) == 4 ? 1 : 2;
  // float of 128: places in LDS worked out anew for each part leave registers enough for a second wave a SIMD
  // (89835 x 9 sharing 3, window 504: 2.18 ms with one, 1.92 ms with two)
  constexpr bool TIGHT = sizeof(T) == 4 && D == 128;
  const int item = item_of_block(tiles * p.heads);
  if (item < 0) return;
  const int group = p.heads / p.kv_heads;
  const int kv = item / (tiles * group), rest = item % (tiles * group);
  const int t0 = rest / group * WA_OWN, head = kv * group + rest % group;
  __shared__ __align__(16) T kt[WA_TILE * D], vt[WA_TILE * D];
  __shared__ int flag[2];
  if (threadIdx.x < 2) flag[threadIdx.x] = 0;
  const QueryRows r = query_rows(p, t0);
  const KeyTiles tl(p, r, t0);
  const int h8 = (lane_id() >> 5) * 8;
  const bool in = r.start <= r.i;
  const int own = p.s.n - t0 < WA_OWN ? p.s.n - t0 : WA_OWN;
  Frag<T> qf[D / 16];
  load_own<T, D, VEC>(qf, p.q, rows_buffer<T, !VEC>(p.q, head, t0, own), r.i - t0, in);
  f32x16 acc[D / 32];
  float m, l;
  const float c = p.scale * kLog2e;
  Staged<T, D, WA_TILE, WA_THREADS, VEC> ks, vs;
  m = -INFINITY;
  l = 0.f;
#pragma unroll
  for (int t = 0; t < D / 32; ++t) acc[t] = zero16();
  ks.load(p.k, kv, tl.first(0), false, tl.rows(0));
  vs.load(p.v, kv, tl.first(0), false, tl.rows(0));
  for (int t = 0; t < tl.count; ++t) {
    const int j0 = tl.first(t), j1 = tl.end(t);
    __syncthreads();
    ks.settle();
    vs.settle();
    ks.store(kt);
    vs.store(vt);
    if (vs.dirty()) flag[t & 1] = 1;
    if (threadIdx.x == 0) flag[(t & 1) ^ 1] = 0;
    __syncthreads();
    // (rows behind part 0 are part 1's; x counts from the tile's first row)
    const int last = min_of(r.i, j1 - 1) - j0;
    const Seen seen = {max_of(r.i - p.window + 1, r.start) - j0, last, r.start - j0, min_of(r.start + p.sinks - 1 - j0, last)};
    if (__builtin_expect(flag[t & 1], 0)) {
      add_not_finite<T, D>(acc, vt, seen);
      __syncthreads();
      vs.clean();
      vs.store(vt);
      __syncthreads();
    }
    if (t + 1 < tl.count) {
      ks.load(p.k, kv, tl.first(t + 1), false, tl.rows(t + 1));
      vs.load(p.v, kv, tl.first(t + 1), false, tl.rows(t + 1));
    }
    if (!r.any(p, j0, WA_TILE)) continue;
    const bool full = r.all && j0 + WA_TILE - 1 <= r.wmin && j0 > r.wmax - p.window && j0 >= r.wstart;
    // Two parts of 32 rows.  The matrix cores work on one part's scores while the weights of the other are taken,
    // and on the products with the first part's weights while those of the second are.
    f32x16 s[2];
    auto scores = [&](int u) __attribute__((always_inline)) {
      s[u] = zero16();
#pragma unroll
      for (int b = 0; b < D / 16; ++b) s[u] = mma(row_frag<D>(kt, u * 32 + pi_of(lane_id() & 31), 16 * b + h8), qf[b], s[u]);
    };
    auto mask = [&](int u) __attribute__((always_inline)) {
      if (!full) {
        asm volatile("");  // (a branch, not selects: most tiles need none)
        if (j0 < r.wstart + p.sinks) mask_part<true>(s[u], seen, u * 32 + h8, -INFINITY);
        else mask_part<false>(s[u], seen, u * 32 + h8, -INFINITY);
      }
    };
    // A new maximum is taken only when some weight would exceed 2^8: the factor cancels in the end.
    auto maximum = [&](const f32x16 &of, bool behind) __attribute__((always_inline)) {
      float top = of[0];
#pragma unroll
      for (int x = 1; x < 16; ++x) top = fmaxf(top, of[x]);
      top = fmaxf(top, other_half(top)) * c;
      if (__any(top > m + 8.f)) {
        // (each row by itself: what other rows of the wave hold does not show in its rounding)
        const bool up = top > m + 8.f;
        const float by = up ? exp2_hw(m - top) : 1.f;
        m = up ? top : m;
        l *= by;
#pragma unroll
        for (int t2 = 0; t2 < D / 32; ++t2)
#pragma unroll
          for (int x = 0; x < 16; ++x) acc[t2][x] *= by;
        if (behind)
#pragma unroll
          for (int x = 0; x < 16; ++x) s[0][x] *= by;  // (weights by now)
      }
    };
    auto weights = [&](int u) __attribute__((always_inline)) {
      const float mm = m > -INFINITY ? m : 0.f;
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        s[u][x] = exp2_hw(__builtin_fmaf(s[u][x], c, -mm));
        l += s[u][x];
      }
    };
    if (PARTS == 1) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (!r.any(p, j0 + u * 32, 32)) continue;
        if constexpr (TIGHT) {
          int l = lane_id();
          asm volatile("" : "+v"(l));
          s[u] = zero16();
#pragma unroll
          for (int b = 0; b < D / 16; ++b) s[u] = mma(row_frag<D>(kt, u * 32 + pi_of(l & 31), 16 * b + (l >> 5) * 8), qf[b], s[u]);
          mask(u);
          maximum(s[u], false);
          weights(u);
          add_rows_at<D>(acc, vt, u * 32, s[u], l);
        } else {
          scores(u);
          mask(u);
          maximum(s[u], false);
          weights(u);
          add_rows<T, D>(acc, vt, u * 32, s[u]);
        }
      }
    } else if (D == 128) {
      constexpr int N = D / 16, VALU = 64 / N;
      scores(0);
      side_by_side<N, 1, 4, 0>();
      mask(0);
      maximum(s[0], false);
      weights(0);
      scores(1);
      side_by_side<N, 1, 4, VALU>();
      hold(s[0]);
      mask(1);
      maximum(s[1], true);
      add_rows<T, D>(acc, vt, 0, s[0]);
      weights(1);
      side_by_side<N, 2, 3, VALU>();
      hold(s[1]);
      add_rows<T, D>(acc, vt, 32, s[1]);
      side_by_side<N, 2, 3, 0>();
    } else {
      // (three waves a SIMD fit: they fill each other's waits, and one maximum serves both parts)
      scores(0);
      scores(1);
      mask(0);
      mask(1);
      f32x16 both;
#pragma unroll
      for (int x = 0; x < 16; ++x) both[x] = fmaxf(s[0][x], s[1][x]);
      maximum(both, false);
      weights(0);
      weights(1);
      add_rows<T, D>(acc, vt, 0, s[0]);
      add_rows<T, D>(acc, vt, 32, s[1]);
    }
  }
  l += other_half(l);
  // a row of no series gets zeros
  const float by = in ? 1.f / l : 0.f;
  store_own<T, D, VEC>(acc, by, p.out, rows_buffer<T>(p.out, head, t0, own), r.i - t0);
  if (p.lse && r.i < p.s.n && lane_id() < 32)
    p.lse[(int64_t)r.i * p.heads + head] = in ? (m + log2_hw(l)) * kLn2 : -INFINITY;
}

// dq, and do.o for the kernel that follows.  Scores are computed again: 6 D operations for each element and no running
// maximum, and 2 D more for the rest of dS.  32768 x 16 x 64, window 1000: 298 us, 780 TFLOP/s with those.  bf16 of 128
// spills 15 registers (25 for rows of odd sizes).
template <typename T, int D, bool VEC>
__global__ __launch_bounds__(WA_THREADS, D * sizeof(T) >= 512 ? 1 : 2) void window_dq_kernel(WindowParams p, int tiles) {
  const int item = item_of_block(tiles * p.heads);
  if (item < 0) return;
  const int group = p.heads / p.kv_heads;
  const int kv = item / (tiles * group), rest = item % (tiles * group);
  const int t0 = rest / group * WA_OWN, head = kv * group + rest % group;
  __shared__ __align__(16) T kt[WA_TILE * D], vt[WA_TILE * D];
  __shared__ int flag[2];
  if (threadIdx.x < 2) flag[threadIdx.x] = 0;
  const QueryRows r = query_rows(p, t0);
  const KeyTiles tl(p, r, t0);
  const int h8 = (lane_id() >> 5) * 8;
  const bool in = r.start <= r.i;
  const int own = p.s.n - t0 < WA_OWN ? p.s.n - t0 : WA_OWN;
  Frag<T> qf[D / 16], of[D / 16];
  load_own<T, D, VEC>(of, p.out, rows_buffer<T, !VEC>(p.out, head, t0, own), r.i - t0, in);
  load_own<T, D, VEC>(qf, p.dout, rows_buffer<T, !VEC>(p.dout, head, t0, own), r.i - t0, in);
  float delta = 0.f;
#pragma unroll
  for (int b = 0; b < D / 16; ++b)
#pragma unroll
    for (int e = 0; e < 8; ++e) delta = __builtin_fmaf((float)of[b][e], (float)qf[b][e], delta);
  delta += other_half(delta);
  if (r.i < p.s.n && lane_id() < 32) p.delta[(int64_t)r.i * p.heads + head] = delta;
#pragma unroll
  for (int b = 0; b < D / 16; ++b) of[b] = qf[b];
  load_own<T, D, VEC>(qf, p.q, rows_buffer<T, !VEC>(p.q, head, t0, own), r.i - t0, in);
  const float lse2 = in ? p.lse[(int64_t)r.i * p.heads + head] * kLog2e : 0.f;
  f32x16 acc[D / 32];
  const float c = p.scale * kLog2e;
  Staged<T, D, WA_TILE, WA_THREADS, VEC> ks, vs;
#pragma unroll
  for (int t = 0; t < D / 32; ++t) acc[t] = zero16();
  ks.load(p.k, kv, tl.first(0), false, tl.rows(0));
  vs.load(p.v, kv, tl.first(0), false, tl.rows(0));
  for (int t = 0; t < tl.count; ++t) {
    const int j0 = tl.first(t), j1 = tl.end(t);
    __syncthreads();
    ks.settle();
    vs.settle();
    ks.store(kt);
    vs.store(vt);
    if (ks.dirty()) flag[t & 1] = 1;
    if (threadIdx.x == 0) flag[(t & 1) ^ 1] = 0;
    __syncthreads();
    // (rows behind part 0 are part 1's; x counts from the tile's first row)
    const int last = min_of(r.i, j1 - 1) - j0;
    const Seen seen = {max_of(r.i - p.window + 1, r.start) - j0, last, r.start - j0, min_of(r.start + p.sinks - 1 - j0, last)};
    if (__builtin_expect(flag[t & 1], 0)) {
      mark_not_finite<T, D>(acc, kt, seen);
      __syncthreads();
      ks.clean();
      ks.store(kt);
      __syncthreads();
    }
    if (t + 1 < tl.count) {
      ks.load(p.k, kv, tl.first(t + 1), false, tl.rows(t + 1));
      vs.load(p.v, kv, tl.first(t + 1), false, tl.rows(t + 1));
    }
    if (!r.any(p, j0, WA_TILE)) continue;
    const bool full = r.all && j0 + WA_TILE - 1 <= r.wmin && j0 > r.wmax - p.window && j0 >= r.wstart;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (!r.any(p, j0 + u * 32, 32)) continue;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int b = 0; b < D / 16; ++b) {
        s = mma(row_frag<D>(kt, u * 32 + pi_of(lane_id() & 31), 16 * b + h8), qf[b], s);
        dp = mma(row_frag<D>(vt, u * 32 + pi_of(lane_id() & 31), 16 * b + h8), of[b], dp);
      }
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const float w = exp2_hw(__builtin_fmaf(s[x], c, -lse2)) * (dp[x] - delta);
        s[x] = w;
      }
      if (!full) {
        asm volatile("");
        if (j0 < r.wstart + p.sinks) mask_part<true>(s, seen, u * 32 + h8, 0.f);
        else mask_part<false>(s, seen, u * 32 + h8, 0.f);
      }
      add_rows<T, D>(acc, kt, u * 32, s);
      if (sizeof(T) == 2) add_rows<T, D>(acc, kt, u * 32, left_over<T>(s));
    }
  }
  store_own<T, D, VEC>(acc, p.scale, p.dq, rows_buffer<T>(p.dq, head, t0, own), r.i - t0);
}

// Last query row + 1 whose pairs with the key rows of tile [j0, j0 + WA_OWN) the main dk/dv kernel adds: the window's.
// Pairs of rows that stay visible with later rows are the sink kernel's.
__device__ inline int last_query(const WindowParams &p, int j0) { return window_end(j0, WA_OWN, p.window, p.s.n); }

// Waves a SIMD of the kernel below, and whether its places in LDS are worked out anew for each part, which frees the
// registers that hold them (float's many matrix instructions leave the time).  Float of 64 gets its second wave so
// (5170 x 28 x 33, window 88: 305 us with one wave, 327 us with one and new places, 311 us with two and old ones, 248 us
// so); float of 128 spills less (7950 x 28 x 128, window 94: 1103 us otherwise, 635 us with tiles of 32 rows besides; its sinks 309 and 256 us).
constexpr bool wa_tight(int bytes, int d) { return bytes == 4 && d >= 64; }
constexpr int wa_waves(int bytes, int d) { return d * bytes < 256 || (d * bytes == 256 && wa_tight(bytes, d)) ? 2 : 1; }

// dk and dv: a block owns key rows and streams the query rows that see them, head after head of the
// group that shares them.  SINK: the rows that stay visible, against the query rows of one section
// that lie beyond what the other form adds; leaves its sums as a part for sink_sum_kernel.
// 32768 x 16 x 64 sharing 4, window 1000: 406 us, 715 TFLOP/s (10 D operations an element); its four sinks 43 us.  Heads
// of 128, window 600: 848 us, one wave a SIMD.
template <typename T, int D, bool VEC, bool SINK>
__global__ __launch_bounds__(WA_THREADS, wa_waves(sizeof(T), D)) void window_dkdv_kernel(WindowParams p, int tiles) {
  constexpr bool TIGHT = wa_tight(sizeof(T), D);
  constexpr int TILE = TIGHT && D == 128 && !SINK ? 32 : WA_TILE;  // (a section's two waves take a part each of 64)
  const int item = item_of_block(tiles * p.kv_heads);
  if (item < 0) return;
  const int group = p.heads / p.kv_heads;
  const int kv = item / tiles, tile = item % tiles;
  const int wave = wave_id(), lane = lane_id(), h8 = (lane >> 5) * 8;
  __shared__ __align__(16) T qt[TILE * D], dt[TILE * D];
  __shared__ float lse_t[TILE], delta_t[TILE];
  __shared__ int flag[2];
  if (threadIdx.x < 2) flag[threadIdx.x] = 0;
  int j, start, end, i0, i1, from = 0;  // the lane's key row and its series; query rows [i0, i1), those before `from` left out
  if (SINK) {
    const int sec0 = tile * WA_SECTION;
    Offsets w = offsets_at(p.s, sec0, false);
    const Span sp = span_of(p.s, w, sec0, false);
    if (sp.index < 0 || sp.start >= sec0) return;  // (uniform) no series reaches over the section's start
    j = sp.start + (lane & 31);
    start = sp.start;
    end = (lane & 31) < p.sinks && j < sp.end ? sp.end : j;
    // a row of this kernel's tile of the other form has pairs up to last_query there
    from = last_query(p, j / WA_OWN * WA_OWN);
    i0 = sec0;
    i1 = sec0 + WA_SECTION < sp.end ? sec0 + WA_SECTION : sp.end;
    if (j / WA_SECTION >= tile) from = i1;  // (a sink row inside the section itself: all its pairs are the other form's)
  } else {
    const int j0 = tile * WA_OWN, j1 = j0 + WA_OWN < p.s.n ? j0 + WA_OWN : p.s.n;
    Offsets w = offsets_at(p.s, j0, false);
    j = j0 + wave * 32 + (lane & 31);
    const Span mine = lane_span(p.s, w, j0, j1 - 1, j);
    const bool in = j < j1 && mine.start <= j;
    start = in ? mine.start : j;
    end = in ? mine.end : j;
    i0 = j0;
    const Span last = span_of(p.s, w, j1 - 1, false);
    i1 = last_query(p, j0);
    const int reach = last.index < 0 ? j1 : last.end;
    if (i1 > reach) i1 = reach;
    if (i1 < j1) i1 = j1;
  }
  const bool in = end > j;
  Frag<T> kf[D / 16], vf[D / 16];
  // the block's own rows, from j_first on (a series' first rows may be fewer than 32)
  const int j_first = SINK ? start : tile * WA_OWN, own = p.s.n - j_first < WA_OWN ? p.s.n - j_first : WA_OWN;
  load_own<T, D, VEC>(kf, p.k, rows_buffer<T, !VEC>(p.k, kv, j_first, own), j - j_first, in);
  load_own<T, D, VEC>(vf, p.v, rows_buffer<T, !VEC>(p.v, kv, j_first, own), j - j_first, in);
  f32x16 dk[D / 32], dv[D / 32];
  const float c = p.scale * kLog2e;
  const int per_head = (i1 - i0 + TILE - 1) / TILE, count = per_head * group;
  Staged<T, D, TILE, WA_THREADS, VEC> qs, ds;
  float lse_n = 0.f, delta_n = 0.f;
  auto fetch = [&](int t) __attribute__((always_inline)) {
    const int head = kv * group + t / per_head, first = i0 + t % per_head * TILE;
    const int rows = i1 - first < TILE ? i1 - first : TILE;
    qs.load(p.q, head, first, false, rows);
    ds.load(p.dout, head, first, false, rows);
    if (threadIdx.x < TILE && (int)threadIdx.x < rows) {
      const int64_t at = (int64_t)(first + threadIdx.x) * p.heads + head;
      lse_n = p.lse[at] * kLog2e;
      delta_n = p.delta[at];
    }
  };
  const int wmin_j = SINK ? start : tile * WA_OWN + wave * 32, wmax_j = wmin_j + 31;
  // of the wave: last series end, first query row of any, and what all have in common
  const int wend = wave_max(end), wfrom = SINK ? wave_max(from) : 0, wfirst = SINK ? wave_min(from) : 0;
  const int wlast = min_of(wave_min(end), i1);
  const bool wall = __all(in), wsink = __any(in && j < start + p.sinks);
#pragma unroll
  for (int t = 0; t < D / 32; ++t) { dk[t] = zero16(); dv[t] = zero16(); }
  if (count > 0) fetch(0);
  for (int t = 0; t < count; ++t) {
    const int r0 = i0 + t % per_head * TILE;
    __syncthreads();
    qs.settle();
    ds.settle();
    qs.store(qt);
    ds.store(dt);
    if (qs.dirty() || ds.dirty()) flag[t & 1] = 1;
    if (threadIdx.x == 0) flag[(t & 1) ^ 1] = 0;
    if (threadIdx.x < TILE) { lse_t[threadIdx.x] = lse_n; delta_t[threadIdx.x] = delta_n; }
    __syncthreads();
    // query rows [first, last] of a tile see key row j: those of its window, all behind it if it stays visible
    const int last = min_of(end, i1) - 1 - r0;
    const Seen seen = {max_of(j, from) - r0, min_of(j < start + p.sinks ? last : window_reach(j, r0, p.window), last), 0, -1};
    if (__builtin_expect(flag[t & 1], 0)) {
      if (!SINK || wave == 0) {  // (two waves share a section's rows: the first speaks for both)
        add_not_finite<T, D, TILE>(dv, dt, seen);
        mark_not_finite<T, D, TILE>(dk, qt, seen);
      }
      __syncthreads();
      qs.clean();
      qs.store(qt);
      ds.clean();
      ds.store(dt);
      __syncthreads();
    }
    if (t + 1 < count) fetch(t + 1);
#pragma unroll
    for (int u = 0; u < TILE / 32; ++u) {
      const int ru = r0 + u * 32;
      if (SINK) {
        if (wave != (ru - i0) / 32 % 2 || ru + 32 <= wfirst) continue;  // two waves share the section's rows
      } else {
        if (ru + 31 < wmin_j || ru >= wend) continue;
        if (!wsink && beyond_window(ru, wmax_j, p.window)) continue;
      }
      int l = lane;
      if (TIGHT) asm volatile("" : "+v"(l));
      const int h = TIGHT ? (l >> 5) * 8 : h8;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int b = 0; b < D / 16; ++b) {
        s = mma(row_frag<D>(qt, u * 32 + pi_of(l & 31), 16 * b + h), kf[b], s);
        dp = mma(row_frag<D>(dt, u * 32 + pi_of(l & 31), 16 * b + h), vf[b], dp);
      }
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int row = u * 32 + 16 * (x >> 3) + h8 + (x & 7);
        s[x] = exp2_hw(__builtin_fmaf(s[x], c, -lse_t[row]));
        dp[x] = s[x] * (dp[x] - delta_t[row]);
      }
      if (!(wall && ru >= wmax_j && ru >= wfrom && ru + 31 < wlast && !beyond_window(ru + 31, wmin_j, p.window))) {
        asm volatile("");
        mask_part<false>(s, seen, u * 32 + h8, 0.f);
        mask_part<false>(dp, seen, u * 32 + h8, 0.f);
      }
      if constexpr (TIGHT) {
        add_rows_at<D>(dv, dt, u * 32, s, l);
        add_rows_at<D>(dk, qt, u * 32, dp, l);
      } else {
        add_rows<T, D>(dv, dt, u * 32, s);
        add_rows<T, D>(dk, qt, u * 32, dp);
        if (sizeof(T) == 2) add_rows<T, D>(dk, qt, u * 32, left_over<T>(dp));
      }
    }
  }
  if (SINK) {
    if (wave > 1) return;
    const int width = p.k.dim + p.v.dim, at = (lane & 31) * width;  // (rows behind the sinks are behind the buffer's end)
    const Buffer o = buffer_of(p.sink_part + (((int64_t)tile * 2 + wave) * p.kv_heads + kv) * p.sinks * width, p.sinks * width * 4);
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int d = t * 32 + 16 * (x >> 3) + h8 + (x & 7);
        const float a = dk[t][x], b = dv[t][x];
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, a), o, d < p.k.dim ? (at + d) * 4 : kOutside, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, b), o, d < p.v.dim ? (at + p.k.dim + d) * 4 : kOutside, 0, 0);
      }
    return;
  }
  const bool more = in && j < start + p.sinks && (end - 1) / WA_SECTION > start / WA_SECTION;
  if (p.sinks > 0 && __any(more)) {
    // what the sections behind the series' first add, summed up in the place of the first of them
    const int width = p.k.dim + p.v.dim;
    const float *o = p.sink_part + (more ? (((int64_t)(start / WA_SECTION + 1) * 2 * p.kv_heads + kv) * p.sinks + (j - start)) * width : 0);
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int d = t * 32 + 16 * (x >> 3) + h8 + (x & 7);
        const bool on_k = more & (d < p.k.dim), on_v = more & (d < p.v.dim);
        const float a = o[on_k ? d : 0], b = o[on_v ? p.k.dim + d : 0];
        dk[t][x] += on_k ? a : 0.f;
        dv[t][x] += on_v ? b : 0.f;
      }
  }
  store_own<T, D, VEC>(dk, p.scale, p.dk, rows_buffer<T>(p.dk, kv, j_first, own), j - j_first);
  store_own<T, D, VEC>(dv, 1.f, p.dv, rows_buffer<T>(p.dv, kv, j_first, own), j - j_first);
}

// Adds up the parts of all sections that a series reaches into, in the place of the first of them.  A
// block takes one (section, key/value head) and has work only where the section is such a first one (13 us there:
// latency, eight sums a thread at a time).
__global__ __launch_bounds__(256) void sink_sum_kernel(WindowParams p) {
  const int sec = blockIdx.x / p.kv_heads, kv = blockIdx.x % p.kv_heads;
  const int sec0 = sec * WA_SECTION;
  Offsets w = offsets_at(p.s, sec0, false);
  const Span sp = span_of(p.s, w, sec0, false);
  if (sp.index < 0 || sp.start >= sec0 || sp.start / WA_SECTION + 1 != sec) return;
  const int last = (sp.end - 1) / WA_SECTION;
  const int count = p.sinks * (p.k.dim + p.v.dim);
  const int64_t step = (int64_t)p.kv_heads * count;  // from one part to the next
  float *o = p.sink_part + ((int64_t)sec * 2 * p.kv_heads + kv) * count;
  for (int e = threadIdx.x; e < count; e += 256) {
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const int parts = (last - sec + 1) * 2;
    int a = 0;
    for (; a + 8 <= parts; a += 8)
#pragma unroll
      for (int x = 0; x < 8; ++x) sum[x] += o[(a + x) * step + e];
    for (; a < parts; ++a) sum[0] += o[a * step + e];
    o[e] = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
  }
}

// ---- host ----------------------------------------------------------------------------------------

static int window_check(const tmp_window_attention_args *a, const char *what, bool grad) {
  TMP_REQUIRE(a != nullptr, TMP_EINVAL, "%s: null args", what);
  TMP_REQUIRE(a->n >= 0 && a->n < (1ll << 31) - 65536, TMP_EINVAL, "%s: row count must be in [0, 2^31 - 65536)", what);
  TMP_SERIES(what, a);
  TMP_REQUIRE(a->type == TMP_BF16 || a->type == TMP_F32, TMP_EUNSUPPORTED, "%s: type must be bfloat16 or float32", what);
  TMP_REQUIRE(a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0 && a->heads <= 65536, TMP_EINVAL,
              "%s: heads (%d) must be a multiple of kv_heads (%d), at most 65536", what, a->heads, a->kv_heads);
  TMP_REQUIRE(a->dim_k > 0 && a->dim_v > 0, TMP_EINVAL, "%s: head sizes must be positive", what);
  TMP_REQUIRE(a->dim_k <= TMP_MAX_HEAD_DIM && a->dim_v <= TMP_MAX_HEAD_DIM, TMP_EUNSUPPORTED,
              "%s: head sizes are limited to %d", what, TMP_MAX_HEAD_DIM);
  TMP_REQUIRE(a->window >= 1, TMP_EINVAL, "%s: window must be >= 1", what);
  TMP_REQUIRE(a->scale > 0.f && a->scale < INFINITY, TMP_EINVAL, "%s: scale must be positive and finite", what);
  TMP_REQUIRE(a->sinks >= 0, TMP_EINVAL, "%s: sinks must be >= 0", what);
  TMP_REQUIRE(a->sinks <= TMP_MAX_SINKS, TMP_EUNSUPPORTED, "%s: at most %d sinks", what, TMP_MAX_SINKS);
  TMP_REQUIRE((a->n + WA_OWN - 1) / WA_OWN * a->heads <= kMostBlocks, TMP_EUNSUPPORTED,
              "%s: too many rows x heads, at most 2^24 - 8 times %d", what, WA_OWN);
  if (a->n == 0) return TMP_OK;
  TMP_REQUIRE(a->q.p && a->k.p && a->v.p && a->out.p, TMP_EINVAL, "%s: null pointer", what);
  if (grad)
    TMP_REQUIRE(a->dout.p && a->dq.p && a->dk.p && a->dv.p && a->lse, TMP_EINVAL, "%s: null pointer", what);
  return TMP_OK;
}

static int window_params(const tmp_window_attention_args *a, const char *what, bool grad, WindowParams *p) {
  memset(p, 0, sizeof(*p));
  const int b = a->type == TMP_F32 ? 4 : 2;
  p->s.offsets = a->offsets; p->s.n_series = a->offsets ? a->n_series : 1; p->s.n = (int32_t)a->n;
  TMP_ROWS(what, a->q, a->n, a->dim_k, b, &p->q);
  TMP_ROWS(what, a->k, a->n, a->dim_k, b, &p->k);
  TMP_ROWS(what, a->v, a->n, a->dim_v, b, &p->v);
  TMP_ROWS(what, a->out, a->n, a->dim_v, b, &p->out);
  if (grad) {
    TMP_ROWS(what, a->dout, a->n, a->dim_v, b, &p->dout);
    TMP_ROWS(what, a->dq, a->n, a->dim_k, b, &p->dq);
    TMP_ROWS(what, a->dk, a->n, a->dim_k, b, &p->dk);
    TMP_ROWS(what, a->dv, a->n, a->dim_v, b, &p->dv);
  }
  p->lse = a->lse;
  p->heads = a->heads; p->kv_heads = a->kv_heads; p->sinks = a->sinks; p->scale = a->scale;
  p->window = (int32_t)(a->window < a->n ? a->window : a->n);
  return TMP_OK;
}

template <typename T, int D, bool VEC> static void window_forward(const WindowParams &p, hipStream_t st) {
  const int tiles = (p.s.n + WA_OWN - 1) / WA_OWN;
  ProfScope ps("window_forward_kernel", st);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(window_forward_kernel<T, D, VEC>), dim3(grid_of_items((int64_t)tiles * p.heads)),
                     dim3(WA_THREADS), 0, st, p, tiles);
}

template <typename T, int D, bool VEC> static void window_grad(const WindowParams &p, hipStream_t st) {
  const int tiles = (p.s.n + WA_OWN - 1) / WA_OWN, sections = (p.s.n + WA_SECTION - 1) / WA_SECTION;
  {
    ProfScope ps("window_dq_kernel", st);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(window_dq_kernel<T, D, VEC>), dim3(grid_of_items((int64_t)tiles * p.heads)),
                       dim3(WA_THREADS), 0, st, p, tiles);
  }
  if (p.sinks > 0 && sections > 1) {
    {
      ProfScope ps("window_dkdv_kernel(sinks)", st);
      hipLaunchKernelGGL(HIP_KERNEL_NAME(window_dkdv_kernel<T, D, VEC, true>), dim3(grid_of_items((int64_t)sections * p.kv_heads)),
                         dim3(WA_THREADS), 0, st, p, sections);
    }
    TMP_LAUNCH(sink_sum_kernel, dim3(sections * p.kv_heads), dim3(256), st, p);
  }
  ProfScope ps("window_dkdv_kernel", st);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(window_dkdv_kernel<T, D, VEC, false>), dim3(grid_of_items((int64_t)tiles * p.kv_heads)),
                     dim3(WA_THREADS), 0, st, p, tiles);
}

struct WindowPlan {
  float *delta, *sink_part;
};
static void window_plan(const tmp_window_attention_args *a, Workspace &ws, WindowPlan *w) {
  const int64_t n = a->n > 0 ? a->n : 1;
  w->delta = ws.take<float>((size_t)n * a->heads);
  const int64_t sections = (n + WA_SECTION - 1) / WA_SECTION;
  w->sink_part = ws.take<float>(a->sinks > 0 && sections > 1
                                    ? (size_t)sections * 2 * a->kv_heads * a->sinks * (a->dim_k + a->dim_v) : 1);
}

}  // namespace tmp

using namespace tmp;

extern "C" int tmp_window_attention(const tmp_window_attention_args *a, void *stream) {
  clear_error();
  TMP_TRY(window_check(a, "tmp_window_attention", false));
  if (a->n == 0) return TMP_OK;
  WindowParams p;
  TMP_TRY(window_params(a, "tmp_window_attention", false, &p));
  const int d = padded_dim(a->dim_k > a->dim_v ? a->dim_k : a->dim_v);
  const bool vec = p.q.vec && p.k.vec && p.v.vec && p.out.vec;
  TMP_BY_FORM(window_forward, a->type, d, vec, p, (hipStream_t)stream);
  TMP_CHECK_HIP(hipGetLastError());
  return TMP_OK;
}

extern "C" size_t tmp_window_attention_grad_workspace_bytes(const tmp_window_attention_args *a) {
  if (!a || window_check(a, "tmp_window_attention_grad", false) != TMP_OK) return 0;
  Workspace ws(nullptr, 0);
  WindowPlan w;
  window_plan(a, ws, &w);
  return ws.off;
}

extern "C" int tmp_window_attention_grad(const tmp_window_attention_args *a, void *workspace, size_t workspace_bytes,
                                         void *stream) {
  clear_error();
  TMP_TRY(window_check(a, "tmp_window_attention_grad", true));
  if (a->n == 0) return TMP_OK;
  WindowParams p;
  TMP_TRY(window_params(a, "tmp_window_attention_grad", true, &p));
  Workspace ws(workspace, workspace_bytes);
  WindowPlan w;
  window_plan(a, ws, &w);
  TMP_REQUIRE(workspace && !ws.overflow(), TMP_EWORKSPACE, "tmp_window_attention_grad: workspace too small");
  p.delta = w.delta;
  p.sink_part = w.sink_part;
  const int d = padded_dim(a->dim_k > a->dim_v ? a->dim_k : a->dim_v);
  const bool vec = p.q.vec && p.k.vec && p.v.vec && p.out.vec && p.dout.vec && p.dq.vec && p.dk.vec && p.dv.vec;
  TMP_BY_FORM(window_grad, a->type, d, vec, p, (hipStream_t)stream);
  TMP_CHECK_HIP(hipGetLastError());
  return TMP_OK;
}
