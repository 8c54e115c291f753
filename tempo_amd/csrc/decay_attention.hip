// Linear attention with a decay for each head over the rows of each series:
//
//   S_i = lambda S_{i-1} + k_i v_i^T      o_i = scale S_i^T q_i      lambda = exp(log_decay[head])
//
// The state is an exponential moving average of the outer products k v^T.  Rows are worked on in parts
// of up to 32 of one series, with r the row's place in the part and X the state before it:
//
//   o_r = scale (lambda^{r+1} X^T q_r + sum_{s<=r} lambda^{r-s} (q_r.k_s) v_s)
//   X  <- lambda^len X + sum_s lambda^{len-1-s} k_s v_s^T
//
// Backward (G_i = scale q_i do_i^T + lambda G_{i+1}, the same recurrence from the last row to the first):
//   dq_i = scale S_i do_i     dk_i = G_i v_i     dv_i = G_i^T k_i     dS_0 = lambda G_1
// are three walks of the same kernel with the roles of the rows exchanged; the walks towards the first
// row keep Y = lambda G, so that o takes lambda^r of it and the update lambda^{len-s}.  The factor `scale` enters S's
// results and G itself: states are what the caller gives and gets, whatever the scale.
//
// The table is cut into sections of rows that are walked side by side.  Where a series reaches over a
// section's start, a first launch walks each section for the state it adds (keys and values only) and a
// second one strings these together (an elementwise scan over the sections); sections that end with a
// series' end, as with sequences of equal length, are skipped by both.
#include <string.h>

#include "row_limits.h"
#include "series_tile.h"

namespace tmp {

// Rows that travel to LDS together: as many as leave the state its registers.
constexpr int da_piece(int bytes, int dk) { return dk * bytes >= 256 ? 32 : 64; }

struct DecayParams {
  Series s;
  Rows q, k, v, out;
  const float *log_decay;
  const float *state_in;  // [n_series][heads][dk][dv]
  float *state_out;
  float *carry;  // [sections][heads][dk][dv]: the state before a section's first row
  int32_t *link;  // [sections]: how carry comes about, see decay_scan_kernel
  int32_t heads, section, sections;
  int32_t alone;  // a section's block walks a series that reaches over its start from that series' first row
  int32_t reverse, transposed;  // walk from the last row; states lie as [dv][dk] of this walk's roles
  float scale;
};

// Walks that are launched together, one to each blockIdx.y: the backward pass's three have the same sections.
struct DecayWalks {
  DecayParams p[3];
};

// lambda^m with m >= 0; lambda may be 0 (log2 = -infinity).
__device__ inline float power(float log2_decay, int m) { return m == 0 ? 1.f : exp2_hw(log2_decay * (float)m); }

// The series that the row at walk position `pos` lies in, in walk positions.  index -1: a stretch of rows
// that belong to none.
__device__ inline Span walk_span(const DecayParams &p, Offsets &w, int pos) {
  const int n = p.s.n;
  Span sp = span_of(p.s, w, p.reverse ? n - 1 - pos : pos, p.reverse);
  if (p.reverse) {
    const int a = n - sp.end;
    sp.end = n - sp.start;
    sp.start = a;
  }
  return sp;
}

// A wave's state: all of dk, 32 of dv.  Tile t's register x is dk = 32 t + 16 (x / 8) + 8 (lane / 32) + x % 8,
// the lane is dv = strip + pi(lane % 32).
__device__ inline uint32_t state_at(int lane, int t, int x, int kd, int vd, bool transposed) {
  const int dk = 32 * t + 16 * (x >> 3) + (lane >> 5) * 8 + (x & 7), dv = (threadIdx.x >> 6) * 32 + pi_of(lane & 31);
  return dk < kd && dv < vd ? (transposed ? dv * kd + dk : dk * vd + dv) * 4 : kOutside;
}
template <int NT> __device__ inline void state_load(f32x16 (&st)[NT], const float *p, int kd, int vd, bool transposed) {
  const Buffer b = buffer_of(p, kd * vd * 4);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    int lane = lane_id();
    asm volatile("" : "+v"(lane));  // (keeps the offsets from being held in registers over the walk)
#pragma unroll
    for (int x = 0; x < 16; ++x)
      st[t][x] = __builtin_bit_cast(float, (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(b, state_at(lane, t, x, kd, vd, transposed), 0, 0));
  }
  // They are waited for here: left to their first use, which lies in the walk's loop, the wait would stand there and be one
  // for the next tile's rows too, part after part (131072 x 16 x 128: 13 % of the walk).
#pragma unroll
  for (int t = 0; t < NT; ++t) asm volatile("" : "+v"(st[t]));
}
template <int NT> __device__ inline void state_store(const f32x16 (&st)[NT], float *p, int kd, int vd, bool transposed) {
  const Buffer b = buffer_of(p, kd * vd * 4);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    int lane = lane_id();
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const float y = st[t][x];  // (a bit cast of the vector's element itself is one of its first element)
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, y), b, state_at(lane, t, x, kd, vd, transposed), 0, 0);
    }
  }
}

// X <- X + K^T diag(w) V for sixteen rows.  The weighted values do not fit bfloat16; they enter as the sum
// of two such numbers, which leave 2^-17 of a term at most, three where the state itself is returned, which leave nothing
// (all 24 bits of it).
template <int D, bool EXACT> __device__ inline void state_add(f32x16 (&st)[D / 32], const __bf16 *kt, int k0, const float *w, bf16x8 v, int) {
  bf16x8 hi, lo;
  f32x8 x;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)v[e] * w[e];
  hi = __builtin_convertvector(x, bf16x8);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] -= (float)hi[e];
  lo = __builtin_convertvector(x, bf16x8);
  bf16x8 rest;
  if (EXACT) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] -= (float)lo[e];
    rest = __builtin_convertvector(x, bf16x8);
  }
#pragma unroll
  for (int t = 0; t < D / 32; ++t) {
    const bf16x8 kf = col_frag<D>(kt, k0, 32 * t);
    st[t] = mma(kf, hi, st[t]);
    st[t] = mma(kf, lo, st[t]);
    if (EXACT) st[t] = mma(kf, rest, st[t]);
  }
}
template <int D, bool EXACT> __device__ inline void state_add(f32x16 (&st)[D / 32], const float *kt, int k0, const float *w, f32x8 v, int l) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= w[e];
#pragma unroll
  for (int t = 0; t < D / 32; ++t) st[t] = mma(col_frag<D>(kt, k0, 32 * t, l), v, st[t]);
}

// Waves a SIMD: two where state, tiles on their way and decays fit 256 registers with next to no spilling.  Float of 128
// fits because its places in LDS are worked out anew for each part (11071 x 15 x 104/80 training: 959 us with one wave,
// 882 us with two).
constexpr int da_waves(int dk, int dv) { return dv < dk ? 1 : 2; }

// OUT: walks a section and writes its rows.  Otherwise: walks the rows of the section that belong to the
// series which goes on behind it, and leaves the state that they make in carry[section + 1].
//
// A wave owns 32 columns of the values and that strip of the state, in registers; the queries', keys' and
// values' tiles (da_piece rows) are shared, the next ones on their way meanwhile.  Rows are worked on in parts of
// SUB, whose decays are the same for every part but a series' last one.  With bfloat16 rows the decayed scores and the
// state itself enter the products that make a row's result as one bfloat16 number each, off by 2^-8 of a term at most (the
// state that is carried, handed on and returned stays in 32 bits): errors of 2.3e-3 against 64 bits, of which rounding the
// result is 1.66e-3; a second product for each would add nearly a third to the walk's matrix instructions.
// Memory bounds it once there are rows enough: 131072 x 16 x 128 bf16 506 us, 4.2 TB/s (states alone 231 us, 4.6 TB/s);
// 50000 x 16 x 64 bf16, the backward pass's three 313 us, 3.9 TB/s; float by its matrix instructions (30011 x 8 x 40/72:
// 150 us).
template <typename T, int DK, int DV, bool VEC, bool OUT, bool EXACT>
__global__ __launch_bounds__(DV * 2, da_waves(DK, DV)) void decay_walk_kernel(DecayWalks w) {
  const DecayParams &p = w.p[blockIdx.y];
  constexpr bool FRESH = DK * sizeof(T) >= 512;
  constexpr int NT = DK / 32, THREADS = DV * 2, SUB = 32, DA_PIECE = da_piece(sizeof(T), DK);
  const int sec = blockIdx.x / p.heads, head = blockIdx.x % p.heads;
  const int lane = lane_id(), l31 = lane & 31, h8 = (lane >> 5) * 8, strip = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 32;
  const int kd = p.k.dim, vd = p.v.dim;
  const int64_t per_state = (int64_t)kd * vd;
  const int sec0 = sec * p.section, sec1 = section_end(sec0, p.section, p.s.n);
  int pos = sec0;
  Span sp;
  Offsets near = {0, -1};  // (nothing is found in it: filled where it is needed)
  if (OUT) near = offsets_at(p.s, p.reverse ? p.s.n - 1 - sec0 : sec0, p.reverse);
  if (!OUT) {
    Offsets last = offsets_at(p.s, p.reverse ? p.s.n - sec1 : sec1 - 1, false);
    sp = walk_span(p, last, sec1 - 1);
    const bool on = sp.index >= 0 && sp.end > sec1;
    if (head == 0 && threadIdx.x == 0) p.link[sec + 1] = !on ? 0 : sp.start < sec0 ? 2 : 1;
    if (!on) return;
    pos = sp.start > sec0 ? sp.start : sec0;
  } else {
    sp = walk_span(p, near, sec0);
    if (p.alone && sp.index >= 0) pos = sp.start;
  }
  extern __shared__ __align__(16) unsigned char smem[];
  T *kt = (T *)smem, *vt = kt + DA_PIECE * DK, *qt = vt + DA_PIECE * DV;
  __shared__ int flag[2];
  if (threadIdx.x < 2) flag[threadIdx.x] = 0;
  const float ld = p.log_decay[head] * kLog2e;
  const int post = p.reverse ? 1 : 0;
  const float scale_out = p.reverse ? 1.f : p.scale, scale_in = p.reverse ? p.scale : 1.f;  // of states' results, of what is added to them
  // Decays that every whole part shares.  TABLE: they lie in LDS, four to a lane at a time, and leave 32 registers to
  // the state (131072 x 16 x 128 bf16: 517 us with two waves a SIMD, 666 us with one); else in registers, which answer
  // sooner (2000 x 4 x 64: 19 us against 23 us).
  constexpr bool TABLE = DK * sizeof(T) >= 256;
  __shared__ f32x4 within[TABLE ? 4 : 1][64];  // scale lambda^{i-j} of a part's rows i and j <= i
  __shared__ f32x4 behind[2][4];               // lambda^{SUB-1-s+post}, with the scale towards the first row
  float wd[16], w_all[SUB / 2];
  if (TABLE) {
    for (int g = threadIdx.x >> 6; g < 4; g += THREADS / 64) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = 16 * (g >> 1) + h8 + 4 * (g & 1) + e;
        x[e] = j <= l31 ? p.scale * power(ld, l31 - j) : 0.f;
      }
      within[g][lane] = x;
    }
    if (threadIdx.x < 32) {
      const int g = (threadIdx.x >> 2) & 3, j = 16 * (g >> 1) + 8 * (threadIdx.x >> 4) + 4 * (g & 1) + (threadIdx.x & 3);
      ((float *)behind)[threadIdx.x] = scale_in * power(ld, SUB - 1 - j + post);
    }
  } else {
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const int j = 16 * (x >> 3) + h8 + (x & 7);
      wd[x] = OUT && j <= l31 ? p.scale * power(ld, l31 - j) : 0.f;
      w_all[x] = scale_in * power(ld, SUB - 1 - j + post);
    }
  }
  const float into = scale_out * power(ld, l31 + 1 - post), fade_all = power(ld, SUB);
  f32x16 st[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) st[t] = zero16();
  bool fresh = true;
  Staged<T, DK, DA_PIECE, THREADS, VEC, true> qs, ks;
  Staged<T, DV, DA_PIECE, THREADS, VEC, true> vs;
  auto fetch = [&](int at, int len) {
    const int64_t first = p.reverse ? (int64_t)p.s.n - 1 - at : at;
    ks.load(p.k, head, first, p.reverse, len);
    vs.load(p.v, head, first, p.reverse, len);
    if (OUT) qs.load(p.q, head, first, p.reverse, len);
  };
  auto length = [&](int at, const Span &s) {
    int e = s.end < sec1 ? s.end : sec1;
    if (at < sec0 && e > sec0) e = sec0;  // (rows before the section are walked for the state only)
    return e - at < DA_PIECE ? e - at : DA_PIECE;
  };
  int len = length(pos, sp), turn = 0;
  fetch(pos, sp.index < 0 ? 0 : len);
  while (true) {
    __syncthreads();
    ks.settle();
    vs.settle();
    ks.store(kt);
    vs.store(vt);
    if (OUT) {
      qs.settle();
      qs.store(qt);
      if (vs.dirty()) flag[turn] = 1;
    }
    if (threadIdx.x == 0) flag[turn ^ 1] = 0;
    __syncthreads();
    const bool dirty = OUT && flag[turn];
    turn ^= 1;
    int bad[2] = {DA_PIECE, DA_PIECE};  // of the lane's column, in either half: the first row that is not finite
    if (__builtin_expect(dirty, 0)) {
#pragma unroll 1
      for (int j = 0; j < DA_PIECE; ++j) {
        const bool on = !finite(tile_elem<T, DV>(vt, j, strip + pi_of(l31)));
        if (j < 32) bad[0] = on && j < bad[0] ? j : bad[0];
        else bad[1] = on && j - 32 < bad[1] ? j - 32 : bad[1];
      }
      __syncthreads();
      vs.clean();  // (a zero weight would not keep such values out of the rows before them)
      vs.store(vt);
      __syncthreads();
    }
    const int next = pos + len;
    Span nsp = sp;
    int nlen = 0;
    if (next < sec1) {
      if (next >= sp.end) nsp = walk_span(p, near, next);
      nlen = length(next, nsp);
      fetch(next, nsp.index < 0 ? 0 : nlen);
    }
    const bool ends = next >= sp.end;
    if (fresh) {
      const float *from = sp.index < 0 ? nullptr
                          : sp.start < pos ? (OUT ? p.carry + ((int64_t)sec * p.heads + head) * per_state : nullptr)
                          : p.state_in ? p.state_in + ((int64_t)sp.index * p.heads + head) * per_state : nullptr;
      if (from) {
        const bool own = sp.start < pos;  // a carry lies as this walk left it
        state_load(st, from, kd, vd, !own && p.transposed);
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) st[t] = zero16();
      }
    }
#pragma unroll 1
    for (int r0 = 0; r0 < len; r0 += SUB) {
      int l = lane;
      if (FRESH) asm volatile("" : "+v"(l));
      const int l31 = l & 31, h8 = (l >> 5) * 8;
      const int rows = len - r0 < SUB ? len - r0 : SUB;
      if (OUT && pos >= sec0) {
        f32x16 acc = zero16(), s = zero16();
#pragma unroll
        for (int b = 0; b < DK / 16; ++b) {
          if (sizeof(T) == 4 && 16 * b >= kd) break;  // (float's instructions are long enough to be worth the branch)
          const Frag<T> qf = row_frag<DK>(qt, r0 + l31, 16 * b + h8);
          s = mma(row_frag<DK>(kt, r0 + pi_of(l31), 16 * b + h8), qf, s);
          acc = mma(operand<T>(st[b >> 1], b & 1), qf, acc);
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          acc[x] *= into;
          s[x] = 16 * (x >> 3) + h8 + (x & 7) <= l31 ? s[x] * (TABLE ? within[x >> 2][lane][x & 3] : wd[x]) : 0.f;
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) acc = mma(col_frag<DV>(vt, r0 + 16 * b, strip, l), operand<T>(s, b), acc);
        if (__builtin_expect(dirty, 0)) {  // they reach the rows at and behind their own, as NaN
          const int first = r0 ? bad[1] : bad[0];
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const int at = __shfl(first, pi_of(16 * (x >> 3) + h8 + (x & 7)));
            acc[x] = at <= l31 ? __uint_as_float(0x7fc00000u) : acc[x];
          }
        }
        const int r = pos + r0;
        const Run o = rows_buffer<T>(p.out, head, p.reverse ? (int64_t)p.s.n - r - rows : r, rows);
        const uint32_t at = (uint32_t)((p.reverse ? rows - 1 - l31 : l31) * (int)p.out.row * (int)sizeof(T));
#pragma unroll
        for (int b = 0; b < 2; ++b)
          // (backwards, rows from `rows` on would start below zero: they have no elements)
          buffer_store8<T>(o, at, strip + 16 * b + h8, VEC || l31 < rows ? p.out.dim : 0, VEC, operand<T>(acc, b));
      }
      if (sp.index < 0 || (ends && r0 + SUB >= len && !p.state_out)) continue;  // no state, or nobody reads it
      const float fade = rows == SUB ? fade_all : power(ld, rows);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 16; ++x) st[t][x] *= fade;
      if (rows == SUB) {
#pragma unroll
        for (int b = 0; b < SUB / 16; ++b) {
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = TABLE ? behind[lane >> 5][2 * b + (e >> 2)][e & 3] : w_all[8 * b + e];
          state_add<DK, EXACT>(st, kt, r0 + 16 * b, w, col_frag<DV>(vt, r0 + 16 * b, strip, l), l);
        }
      } else {
#pragma unroll 1
        for (int b = 0; 16 * b < rows; ++b) {
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int left = rows - 1 - (16 * b + h8 + e);
            w[e] = left >= 0 ? scale_in * power(ld, left + post) : 0.f;
          }
          state_add<DK, EXACT>(st, kt, r0 + 16 * b, w, col_frag<DV>(vt, r0 + 16 * b, strip, l), l);
        }
      }
      if (__builtin_expect(dirty, 0)) {
        const float x = (r0 ? bad[1] : bad[0]) < DA_PIECE ? __uint_as_float(0x7fc00000u) : 0.f;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int y = 0; y < 16; ++y) st[t][y] += x;
      }
    }
    if (OUT && ends && sp.index >= 0 && p.state_out)
      state_store(st, p.state_out + ((int64_t)sp.index * p.heads + head) * per_state, kd, vd, p.transposed);
    fresh = ends;
    if (next >= sec1) break;
    pos = next;
    len = nlen;
    sp = nsp;
  }
  if (!OUT) state_store(st, p.carry + ((int64_t)(sec + 1) * p.heads + head) * per_state, kd, vd, false);
}

// carry[s] holds what section s - 1 adds; link[s] = 2: all of that section is the one series that goes on
// into s, so that the state before it goes on too, lambda^section times.  A wave strings DA_RUN sections of 64
// elements together, x -> m x + y, the waves of a block theirs through LDS: one trip to memory in place of one
// for every run of sections (64074 rows x 4 x 12, 501 sections: 22 us, 58 us by one wave).
constexpr int DA_RUN = 16, DA_SCAN_WAVES = 16;
__global__ __launch_bounds__(DA_SCAN_WAVES * 64) void decay_scan_kernel(DecayWalks walks, int64_t per_head) {
  const DecayParams &p = walks.p[blockIdx.y];
  const int64_t blocks = (per_head + 63) / 64;
  const int head = (int)(blockIdx.x / blocks), lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t e = (blockIdx.x % blocks) * 64 + lane;
  const bool on = e < per_head;
  const float fade = power(p.log_decay[head] * kLog2e, p.section);
  float *c = p.carry + (int64_t)head * per_head + (on ? e : 0);
  const int64_t step = (int64_t)p.heads * per_head;
  __shared__ float run_add[2][DA_SCAN_WAVES][64], run_fade[2][DA_SCAN_WAVES];
  float x = 0.f;  // the state before the sweep
  for (int s0 = 1, turn = 0; s0 < p.sections; s0 += DA_RUN * waves, turn ^= 1) {
    const int s = s0 + wave * DA_RUN;
    float add[DA_RUN], m = 1.f, y = 0.f;
    int link[DA_RUN];
#pragma unroll
    for (int a = 0; a < DA_RUN; ++a) {
      const int at = s + a < p.sections ? s + a : p.sections - 1;
      link[a] = s + a < p.sections ? p.link[at] : 0;
      add[a] = c[at * step];  // (also where nothing goes on: what lies there is not used then)
    }
    auto next = [&](int a, float before) {
      return link[a] == 2 ? __builtin_fmaf(fade, before, add[a]) : link[a] ? add[a] : 0.f;
    };
#pragma unroll
    for (int a = 0; a < DA_RUN; ++a) {
      y = next(a, y);
      m = link[a] != 2 || m < 0.f ? -1.f : m * fade;  // (below zero: what was before is gone, NaN too)
    }
    run_add[turn][wave][lane] = y;
    if (lane == 0) run_fade[turn][wave] = m;
    __syncthreads();
    float before = 0.f;
    for (int w = 0; w < waves; ++w) {
      if (w == wave) before = x;
      const float by = run_fade[turn][w], plus = run_add[turn][w][lane];
      x = by < 0.f ? plus : __builtin_fmaf(by, x, plus);
    }
#pragma unroll
    for (int a = 0; a < DA_RUN; ++a) {
      before = next(a, before);
      if (on && link[a] == 2) c[(s + a) * step] = before;
    }
  }
}

// A series without rows keeps its state.
__global__ __launch_bounds__(256) void decay_empty_kernel(DecayParams p, int64_t n_series, int64_t per_series) {
  for (int64_t s = blockIdx.x; s < n_series; s += gridDim.x) {
    int64_t a = 0, b = p.s.n;
    if (p.s.offsets) { a = p.s.offsets[s]; b = p.s.offsets[s + 1]; }
    if (b > p.s.n) b = p.s.n;
    if (a < 0) a = 0;
    if (a < b) continue;
    for (int64_t e = threadIdx.x; e < per_series; e += 256)
      p.state_out[s * per_series + e] = p.state_in ? p.state_in[s * per_series + e] : 0.f;
  }
}

// ---- host ----------------------------------------------------------------------------------------

// Sections of whole pieces, as few as give the 1024 SIMDs the two waves each that they hold (a block has one for 32 of
// dv): every one more adds a state to be written, strung together and read.  131072 x 16 x 128 bf16: 256 blocks 1057 us,
// 512 829 us, 1024 860 us, 2048 921 us; training of 50000 x 16 x 64: 512 blocks 544 us, 1024 539 us, 2048 609 us; 30011 x
// 8 x 40/72 float: 256 blocks 253 us, 512 219 us, 1024 227 us.
static int decay_section(int64_t n, int heads, int dim) {
  const int dv = padded_dim(dim);  // the larger of the two sizes: either is the values' in some walk
  const int blocks = 2048 / (dv / 32);
  int64_t s = (n * heads + blocks - 1) / blocks;
  if (s > n) s = n;
  s = (s + 63) / 64 * 64;
  if (s < 64) s = 64;
  return (int)s;
}

struct DecayPlan {
  float *carry;
  int32_t *link;
  int section, sections;
  size_t per_walk;  // floats of carry
};
static void decay_plan(const tmp_decay_attention_args *a, int walks, Workspace &ws, DecayPlan *d) {
  const int64_t n = a->n > 0 ? a->n : 1;
  d->section = decay_section(n, a->heads, a->dim_k > a->dim_v ? a->dim_k : a->dim_v);
  d->sections = (int)((n + d->section - 1) / d->section);
  d->per_walk = d->sections > 1 ? (size_t)d->sections * a->heads * a->dim_k * a->dim_v : 0;  // (nothing is carried)
  d->carry = ws.take<float>(d->per_walk * walks);
  d->link = ws.take<int32_t>((size_t)(d->sections + 1) * walks);
}

static int decay_check(const tmp_decay_attention_args *a, const char *what, bool grad) {
  TMP_REQUIRE(a != nullptr, TMP_EINVAL, "%s: null args", what);
  TMP_REQUIRE(a->n >= 0 && a->n < (1ll << 31) - 65536, TMP_EINVAL, "%s: row count must be in [0, 2^31 - 65536)", what);
  TMP_SERIES(what, a);
  TMP_REQUIRE(a->type == TMP_BF16 || a->type == TMP_F32, TMP_EUNSUPPORTED, "%s: type must be bfloat16 or float32", what);
  TMP_REQUIRE(a->heads > 0 && a->heads <= 65536, TMP_EINVAL, "%s: heads must be in [1, 65536]", what);
  TMP_REQUIRE(a->dim_k > 0 && a->dim_v > 0, TMP_EINVAL, "%s: head sizes must be positive", what);
  TMP_REQUIRE(a->dim_k <= TMP_MAX_HEAD_DIM && a->dim_v <= TMP_MAX_HEAD_DIM, TMP_EUNSUPPORTED,
              "%s: head sizes are limited to %d", what, TMP_MAX_HEAD_DIM);
  TMP_REQUIRE(a->scale > 0.f && a->scale < INFINITY, TMP_EINVAL, "%s: scale must be positive and finite", what);
  if (a->n == 0) return TMP_OK;
  TMP_REQUIRE(a->log_decay && a->q.p && a->k.p && a->v.p, TMP_EINVAL, "%s: null pointer", what);
  if (grad) TMP_REQUIRE(a->dout.p && a->dq.p && a->dk.p && a->dv.p, TMP_EINVAL, "%s: null pointer", what);
  else TMP_REQUIRE(a->out.p, TMP_EINVAL, "%s: null pointer", what);
  return TMP_OK;
}

template <typename T, int DK, int DV, bool VEC, bool EXACT> static void decay_walk(const DecayWalks &w, int walks, hipStream_t st) {
  const DecayParams &p = w.p[0];
  const int threads = DV * 2, row = da_piece(sizeof(T), DK) * (int)sizeof(T);
  if (p.sections > 1 && !p.alone) {
    {
      ProfScope ps("decay_walk_kernel(states)", st);
      hipLaunchKernelGGL(HIP_KERNEL_NAME(decay_walk_kernel<T, DK, DV, VEC, false, EXACT>), dim3((p.sections - 1) * p.heads, walks),
                         dim3(threads), row * (DK + DV), st, w);
    }
    const int64_t per_head = (int64_t)p.k.dim * p.v.dim;
    const int waves = (p.sections + DA_RUN - 2) / DA_RUN;
    TMP_LAUNCH(decay_scan_kernel, dim3((unsigned)((per_head + 63) / 64 * p.heads), walks),
               dim3((waves < DA_SCAN_WAVES ? waves : DA_SCAN_WAVES) * 64), st, w, per_head);
  }
  ProfScope ps("decay_walk_kernel", st);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(decay_walk_kernel<T, DK, DV, VEC, true, EXACT>), dim3(p.sections * p.heads, walks),
                     dim3(threads), row * (2 * DK + DV), st, w);
}
template <typename T, int DK, int DV> static void decay_walk_form(const DecayWalks &w, int walks, hipStream_t st) {
  bool vec = true;
  for (int i = 0; i < walks; ++i) vec = vec && w.p[i].q.vec && w.p[i].k.vec && w.p[i].v.vec && w.p[i].out.vec;
  constexpr bool SPLIT = sizeof(T) == 2;
  if (SPLIT && w.p[0].state_out) {
    if (vec) decay_walk<T, DK, DV, true, SPLIT>(w, walks, st);
    else decay_walk<T, DK, DV, false, SPLIT>(w, walks, st);
  } else {
    if (vec) decay_walk<T, DK, DV, true, false>(w, walks, st);
    else decay_walk<T, DK, DV, false, false>(w, walks, st);
  }
}
// Both head sizes padded to 32, 64 or 128, and at most a factor of two apart.
template <typename T> static void decay_walk_dims(const DecayWalks &w, int walks, hipStream_t st) {
  const DecayParams &p = w.p[0];
  int dk = padded_dim(p.k.dim), dv = padded_dim(p.v.dim);
  if (dk < dv / 2) dk = dv / 2;
  if (dv < dk / 2) dv = dk / 2;
  if (dk == 32) {
    if (dv == 32) decay_walk_form<T, 32, 32>(w, walks, st);
    else decay_walk_form<T, 32, 64>(w, walks, st);
  } else if (dk == 64) {
    if (dv == 32) decay_walk_form<T, 64, 32>(w, walks, st);
    else if (dv == 64) decay_walk_form<T, 64, 64>(w, walks, st);
    else decay_walk_form<T, 64, 128>(w, walks, st);
  } else {
    if (dv == 64) decay_walk_form<T, 128, 64>(w, walks, st);
    else decay_walk_form<T, 128, 128>(w, walks, st);
  }
}
// `walks` of w, all of the same padded head sizes and with a state returned by all or none.
static void decay_run(const DecayWalks &w, int walks, int type, hipStream_t st) {
  if (type == TMP_F32) decay_walk_dims<float>(w, walks, st);
  else decay_walk_dims<__bf16>(w, walks, st);
}

static DecayParams decay_params(const tmp_decay_attention_args *a, const DecayPlan &d, int walk) {
  DecayParams p;
  memset(&p, 0, sizeof(p));
  p.s.offsets = a->offsets; p.s.n_series = a->offsets ? a->n_series : 1; p.s.n = (int32_t)a->n;
  p.log_decay = a->log_decay;
  p.carry = d.carry + walk * d.per_walk; p.link = d.link + walk * (d.sections + 1); p.section = d.section; p.sections = d.sections;
  // Few rows: one launch, whose blocks walk the rows of their first series that lie before them once more, costs less than
  // three.  Lengths are known on the device only, so the bound is where one block's walk over all rows still takes no longer
  // than the three (us of a call, one series of all rows among empty ones | series of 20 rows; one launch, three launches):
  // bf16 4 x 64/64 512 rows 21, 21 | 13, 24, 1024 rows 37, 23 | 13, 26; 16 x 128/128 512 rows 31, 34 | 15, 33, 1024 rows
  // 57, 39 | 15, 35; float 8 x 40/72 256 rows 27, 29 | 23, 32, 512 rows 45, 30 | 23, 33; 2 x 128/128 256 rows 44, 44 | 37, 50.
  p.alone = a->n <= (a->type == TMP_BF16 ? 512 : 256);
  p.heads = a->heads; p.scale = a->scale;
  return p;
}

static int decay_empty(const DecayParams &p, int64_t n_series, int64_t per_series, hipStream_t st) {
  if (p.state_out && n_series > 0)
    TMP_LAUNCH(decay_empty_kernel, dim3((unsigned)(n_series < 65536 ? n_series : 65536)), dim3(256), st, p, n_series, per_series);
  return TMP_OK;
}

}  // namespace tmp

using namespace tmp;

extern "C" size_t tmp_decay_attention_workspace_bytes(const tmp_decay_attention_args *a) {
  // (what the call itself refuses needs none: no more is taken for it than for a call that runs)
  if (!a || a->n < 0 || a->n >= (1ll << 31) - 65536 || a->heads < 1 || a->heads > 65536 || a->dim_k < 1 || a->dim_v < 1 ||
      a->dim_k > TMP_MAX_HEAD_DIM || a->dim_v > TMP_MAX_HEAD_DIM)
    return 0;
  Workspace ws(nullptr, 0);
  DecayPlan d;
  decay_plan(a, a->dout.p || a->n <= 0 ? 3 : 1, ws, &d);  // (without rows there may be no pointers)
  return ws.off;
}

extern "C" int tmp_decay_attention(const tmp_decay_attention_args *a, void *workspace, size_t workspace_bytes, void *stream) {
  clear_error();
  TMP_TRY(decay_check(a, "tmp_decay_attention", false));
  Workspace ws(workspace, workspace_bytes);
  DecayPlan d;
  decay_plan(a, 1, ws, &d);
  TMP_REQUIRE(workspace && !ws.overflow(), TMP_EWORKSPACE, "tmp_decay_attention: workspace too small");
  hipStream_t st = (hipStream_t)stream;
  const int b = a->type == TMP_F32 ? 4 : 2;
  DecayWalks w = {};
  DecayParams &p = w.p[0];
  p = decay_params(a, d, 0);
  const char *what = "tmp_decay_attention";
  if (a->n > 0) {
    TMP_ROWS(what, a->q, a->n, a->dim_k, b, &p.q);
    TMP_ROWS(what, a->k, a->n, a->dim_k, b, &p.k);
    TMP_ROWS(what, a->v, a->n, a->dim_v, b, &p.v);
    TMP_ROWS(what, a->out, a->n, a->dim_v, b, &p.out);
  }
  p.state_in = a->state_in; p.state_out = a->state_out;
  if (a->n > 0) decay_run(w, 1, a->type, st);
  TMP_TRY(decay_empty(p, p.s.n_series, (int64_t)a->heads * a->dim_k * a->dim_v, st));
  TMP_CHECK_HIP(hipGetLastError());
  return TMP_OK;
}

extern "C" int tmp_decay_attention_grad(const tmp_decay_attention_args *a, void *workspace, size_t workspace_bytes, void *stream) {
  clear_error();
  TMP_TRY(decay_check(a, "tmp_decay_attention_grad", true));
  Workspace ws(workspace, workspace_bytes);
  DecayPlan d;
  decay_plan(a, 3, ws, &d);
  TMP_REQUIRE(workspace && !ws.overflow(), TMP_EWORKSPACE, "tmp_decay_attention_grad: workspace too small");
  hipStream_t st = (hipStream_t)stream;
  const int b = a->type == TMP_F32 ? 4 : 2;
  const char *what = "tmp_decay_attention_grad";
  Rows q = {}, k = {}, v = {}, o = {}, dq = {}, dk = {}, dv = {};
  if (a->n > 0) {
    TMP_ROWS(what, a->q, a->n, a->dim_k, b, &q);
    TMP_ROWS(what, a->k, a->n, a->dim_k, b, &k);
    TMP_ROWS(what, a->v, a->n, a->dim_v, b, &v);
    TMP_ROWS(what, a->dout, a->n, a->dim_v, b, &o);
    TMP_ROWS(what, a->dq, a->n, a->dim_k, b, &dq);
    TMP_ROWS(what, a->dk, a->n, a->dim_k, b, &dk);
    TMP_ROWS(what, a->dv, a->n, a->dim_v, b, &dv);
  }
  // The three walks do not depend on each other: those whose kernel is the same go in one launch
  // (training of 24184 x 1 x 84/104: 224 us with three, 158 us so; of 50000 x 16 x 64: 605 us and 555 us).
  DecayWalks w = {};
  for (int i = 0; i < 3; ++i) w.p[i] = decay_params(a, d, i);
  DecayParams &p0 = w.p[0], &p1 = w.p[1], &p2 = w.p[2];
  p0.q = o; p0.k = v; p0.v = k; p0.out = dq;
  p0.state_in = a->state_in; p0.transposed = 1;
  p1.q = v; p1.k = o; p1.v = q; p1.out = dk; p1.transposed = 1;
  p2.q = k; p2.k = q; p2.v = o; p2.out = dv;
  for (int i = 1; i < 3; ++i) { w.p[i].reverse = 1; w.p[i].state_in = a->dstate_out; }
  p2.state_out = a->dstate_in;
  if (a->n > 0) {
    const bool one = !p2.state_out && padded_dim(a->dim_k) == padded_dim(a->dim_v);
    decay_run(w, one ? 3 : 2, a->type, st);
    if (!one) {
      DecayWalks last = {};
      last.p[0] = p2;
      decay_run(last, 1, a->type, st);
    }
  }
  TMP_TRY(decay_empty(p2, p2.s.n_series, (int64_t)a->heads * a->dim_k * a->dim_v, st));
  TMP_CHECK_HIP(hipGetLastError());
  return TMP_OK;
}
