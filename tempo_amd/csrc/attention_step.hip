// Single rows of the two attentions over series: a serving process keeps one slot of state for each
// series and gives, call after call, one new row for some of the slots.
//
// Decay: the state [dk][dv] of a slot is read once, updated and written once -- 8 bytes of traffic and
// five operations an element, so the memory's rate bounds it.
// Window: the cache of a slot holds its first `sinks` rows and a ring of the last `window` others; every
// row in it is visible and their order does not matter, so no mask is needed.  It is read once for all
// query heads that share a key/value head (they are the columns of the matrix cores' result).
//
// slots[b] names the slot of row b.  A row whose slot is out of range or has been named by an earlier row
// of the call changes nothing and results in NaN.
#include <string.h>

#include "series_tile.h"

namespace tmp {

// The slot of row b, -1 if it has none of its own.  All threads of the wave call this together.  Every block looks through
// the slots of the rows before its own: nothing to speak of up to 512 rows, but a decay step of 4096 rows x 16 x 64 takes
// 678 us with slots and 378 without, of the most rows (65536 x 8 x 32) 31 and 1.9 ms.
__device__ inline int slot_of(const int32_t *slots, int b, int n_slots) {
  if (!slots) return b;
  const int s = slots[b];
  bool taken = false;
  for (int i = lane_id(); i < b; i += 64) taken |= slots[i] == s;
  return s < 0 || s >= n_slots || __any(taken) ? -1 : s;
}

struct DecayStepParams {
  Rows q, k, v, out;
  const float *log_decay;
  float *state;
  const int32_t *slots;
  int32_t n, n_slots, heads;
  float scale;
};

// A block takes one (row, head).  Each thread owns VEC neighbouring dv of every (256 / columns)-th dk, sixteen loads in
// flight.  512 x 16 x 128: 218 us, 4.96 TB/s of states read and written; 100 x 8 x 64: 9 us, less than the host's part.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void decay_step_kernel(DecayStepParams p) {
  typedef float fv __attribute__((ext_vector_type(VEC)));
  const int b = blockIdx.x / p.heads, head = blockIdx.x % p.heads;
  const int kd = p.k.dim, vd = p.v.dim;
  __shared__ float qk[2][TMP_MAX_HEAD_DIM];
  __shared__ float part[256 * VEC];
  const T *qp = head_of<T>(p.q, head) + (int64_t)b * p.q.row, *kp = head_of<T>(p.k, head) + (int64_t)b * p.k.row;
  const T *vp = head_of<T>(p.v, head) + (int64_t)b * p.v.row;
  T *op = (T *)p.out.p + (int64_t)head * p.out.head + (int64_t)b * p.out.row;
  if ((int)threadIdx.x < kd) {
    qk[0][threadIdx.x] = (float)qp[threadIdx.x];
    qk[1][threadIdx.x] = (float)kp[threadIdx.x];
  }
  const int slot = slot_of(p.slots, b, p.n_slots);
  __syncthreads();
  const int columns = (vd + VEC - 1) / VEC, per = 256 / columns;
  const int c = threadIdx.x % columns, r = threadIdx.x / columns;
  fv o;
#pragma unroll
  for (int e = 0; e < VEC; ++e) o[e] = 0.f;
  if (slot >= 0 && r < per) {
    const float fade = exp2_hw(p.log_decay[head] * kLog2e);
    float *s = p.state + ((int64_t)slot * p.heads + head) * kd * vd + c * VEC;
    fv v;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (float)vp[c * VEC + e];
    constexpr int AHEAD = 16;
    for (int k0 = r; k0 < kd; k0 += per * AHEAD) {
      fv x[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a)
        if (k0 + a * per < kd) x[a] = *(const fv *)(s + (k0 + a * per) * vd);
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int k = k0 + a * per;
        if (k < kd) {
          const float kk = qk[1][k], qq = qk[0][k];
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            x[a][e] = __builtin_fmaf(fade, x[a][e], kk * v[e]);
            o[e] = __builtin_fmaf(qq, x[a][e], o[e]);
          }
          *(fv *)(s + k * vd) = x[a];
        }
      }
    }
  }
  *(fv *)(part + threadIdx.x * VEC) = o;
  __syncthreads();
  for (int d = threadIdx.x; d < vd; d += 256) {
    float sum = 0.f;
    for (int i = 0; i < per; ++i) sum += part[(i * columns + d / VEC) * VEC + d % VEC];
    op[d] = (T)(slot < 0 ? __uint_as_float(0x7fc00000u) : sum * p.scale);
  }
}

struct WindowStepParams {
  Rows q, k, v, out;   // the new rows
  Rows kc, vc;         // the cache: Rows of one slot
  int64_t kc_slot, vc_slot;
  int64_t *length;
  const int32_t *slots;
  float *part;  // [n][heads][splits][dim_v + 2]: sum of weighted values, maximum, sum of weights
  int32_t n, n_slots, heads, kv_heads, window, sinks, splits, chunk;
  float scale;
};

__device__ inline int place_of(int64_t t, int sinks, int window) {
  return t < sinks ? (int)t : sinks + (int)((t - sinks) % window);
}

// A wave takes `chunk` rows of one slot's cache, one key/value head and up to 32 of its query heads.  Memory bounds it:
// 256 x 32 x 128 sharing 8, window 1000: 182 us, 5.4 TB/s; 9 x 8 x 64 sharing 2, window 600: 9 us of latency.
template <typename T, int D, bool VEC>
__global__ __launch_bounds__(256, D * sizeof(T) >= 512 ? 1 : 2) void window_step_kernel(WindowStepParams p, int units) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (unit >= units) return;
  T *vt = (T *)smem + (threadIdx.x >> 6) * 32 * D;
  const int lane = lane_id(), l31 = lane & 31, h8 = (lane >> 5) * 8;
  const int group = p.heads / p.kv_heads, parts = (group + 31) / 32;
  int u = unit;
  const int split = u % p.splits; u /= p.splits;
  const int part = u % parts; u /= parts;
  const int kv = u % p.kv_heads, b = u / p.kv_heads;
  const int head = kv * group + part * 32 + l31;
  const bool on = part * 32 + l31 < group;
  // What does not depend on the slot is asked for first: a small call is a chain of trips to memory (9 rows x 8 heads
  // sharing 2, window 600: 9.2 -> 9.0 us, its join, which does the same, 6.8 -> 6.4 us).
  Frag<T> qf[D / 16];
  const T *qp = head_of<T>(p.q, on ? head : 0) + (int64_t)b * p.q.row;
#pragma unroll
  for (int x = 0; x < D / 16; ++x)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = 16 * x + h8 + e;
      qf[x][e] = on && d < p.q.dim ? qp[d] : (T)0.f;
    }
  const T *kn = head_of<T>(p.k, kv) + (int64_t)b * p.k.row, *vn = head_of<T>(p.v, kv) + (int64_t)b * p.v.row;
  T new_k[2], new_v[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = lane + 64 * i;
    new_k[i] = kn[d < p.k.dim ? d : 0];
    new_v[i] = vn[d < p.v.dim ? d : 0];
  }
  const int slot = slot_of(p.slots, b, p.n_slots);
  if (slot < 0) return;
  const int64_t t = p.length[slot];
  const int cap = p.window + p.sinks;
  const int count = t < 0 ? 1 : t + 1 < cap ? (int)t + 1 : cap, place = t < 0 ? 0 : place_of(t, p.sinks, p.window);
  const int r0 = split * p.chunk, r1 = r0 + p.chunk < count ? r0 + p.chunk : count;
  float *out = p.part + (((int64_t)b * p.heads + (on ? head : kv * group)) * p.splits + split) * (p.v.dim + 2);
  Rows kc = p.kc, vc = p.vc;
  kc.p = (T *)p.kc.p + slot * p.kc_slot;
  vc.p = (T *)p.vc.p + slot * p.vc_slot;
  // The new row goes into the cache first.  Only the waves whose rows hold its place read that place (waves of
  // the same rows and other query heads write the same there), each behind its own write.
  if (place >= r0 && place < r1) {
    T *ko = (T *)head_of<T>(kc, kv) + (int64_t)place * kc.row, *vo = (T *)head_of<T>(vc, kv) + (int64_t)place * vc.row;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = lane + 64 * i;
      if (d < p.k.dim) ko[d] = new_k[i];
      if (d < p.v.dim) vo[d] = new_v[i];
    }
    __threadfence_block();
  }
  f32x16 acc[D / 32];
#pragma unroll
  for (int x = 0; x < D / 32; ++x) acc[x] = zero16();
  float m = -INFINITY, l = 0.f;
  const float c = p.scale * kLog2e;
  Frag<T> kf[D / 16];
  Staged<T, D, 32, 64, VEC> vs;
  auto fetch = [&](int row0) {
    const int rows = r1 - row0 < 32 ? r1 - row0 : 32;
    const Run kb = rows_buffer<T, !VEC>(kc, kv, row0, rows);  // (what rows behind the last read is masked below)
    const uint32_t at = pi_of(l31) * (uint32_t)kc.row * (uint32_t)sizeof(T);
#pragma unroll
    for (int x = 0; x < D / 16; ++x) kf[x] = buffer_load8<T>(kb, at, 16 * x + h8, kc.dim, VEC);
    vs.load(vc, kv, row0, false, rows);
  };
  if (r0 < r1) fetch(r0);
  for (int row0 = r0; row0 < r1; row0 += 32) {
    f32x16 s = zero16();
#pragma unroll
    for (int x = 0; x < D / 16; ++x) s = mma(kf[x], qf[x], s);
    vs.settle();
    vs.store(vt);
    if (row0 + 32 < r1) fetch(row0 + 32);
    __builtin_amdgcn_wave_barrier();
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      if (row0 + 16 * (x >> 3) + h8 + (x & 7) >= r1) s[x] = -INFINITY;
      top = fmaxf(top, s[x]);
    }
    top = fmaxf(top, other_half(top)) * c;
    const float nm = fmaxf(m, top), by = nm > -INFINITY ? exp2_hw(m - nm) : 1.f, mm = nm > -INFINITY ? nm : 0.f;
    m = nm;
    l *= by;
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      s[x] = exp2_hw(__builtin_fmaf(s[x], c, -mm));
      l += s[x];
    }
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
      for (int y = 0; y < 16; ++y) acc[x][y] *= by;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const Frag<T> hi = operand<T>(s, y);
      Frag<T> lo = hi;
      if (sizeof(T) == 2) {  // what the rounding of the weights leaves goes in as well: the matrix cores have time
        f32x16 rest = s;
#pragma unroll
        for (int e = 0; e < 8; ++e) rest[8 * y + e] -= (float)hi[e];
        lo = operand<T>(rest, y);
      }
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        const Frag<T> f = col_frag<D>(vt, 16 * y, x * 32);
        acc[x] = mma(f, hi, acc[x]);
        if (sizeof(T) == 2) acc[x] = mma(f, lo, acc[x]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  l += other_half(l);
  if (!on) return;
#pragma unroll
  for (int x = 0; x < D / 32; ++x)
#pragma unroll
    for (int y = 0; y < 16; ++y) {
      const int d = x * 32 + 16 * (y >> 3) + h8 + (y & 7);
      if (d < p.v.dim) out[d] = acc[x][y];
    }
  if (lane < 32) {
    out[p.v.dim] = m;
    out[p.v.dim + 1] = l;
  }
}

// Joins the parts of a (row, head); the first head's block counts the row.  A launch of its own (7-12 us) because all parts
// of a slot have read its length by then.
constexpr int WS_MOST_SPLITS = 2048;
template <typename T>
__global__ __launch_bounds__(128) void window_join_kernel(WindowStepParams p) {
  __shared__ float by[WS_MOST_SPLITS];
  const int b = blockIdx.x / p.heads, head = blockIdx.x % p.heads, d = threadIdx.x, lane = lane_id();
  const int slot = slot_of(p.slots, b, p.n_slots);
  T *o = (T *)p.out.p + (int64_t)head * p.out.head + (int64_t)b * p.out.row;
  const int width = p.v.dim + 2;
  const float *in = p.part + ((int64_t)b * p.heads + head) * p.splits * width;
  if (slot < 0) {
    if (d < p.v.dim) o[d] = (T)__uint_as_float(0x7fc00000u);
    return;
  }
  const int64_t seen = head == 0 && d == 0 ? p.length[slot] : 0;  // (early: it is only needed at the end)
  constexpr int FIRST = 8;
  float first[FIRST];  // likewise the first parts' values
#pragma unroll
  for (int a = 0; a < FIRST; ++a) first[a] = in[(a < p.splits ? a : 0) * width + (d < p.v.dim ? d : 0)];
  float top = -INFINITY;
  for (int s = lane; s < p.splits; s += 64) top = fmaxf(top, in[s * width + p.v.dim]);
#pragma unroll
  for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
  const float mm = top > -INFINITY ? top : 0.f;
  float weights = 0.f;
  for (int s = lane; s < p.splits; s += 64) {
    const float e = exp2_hw(in[s * width + p.v.dim] - mm);
    weights = __builtin_fmaf(e, in[s * width + p.v.dim + 1], weights);
    by[s] = e;  // (both waves write the same)
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) weights += __shfl_xor(weights, x);
  __syncthreads();
  if (d < p.v.dim) {
    float sum = 0.f;
#pragma unroll
    for (int a = 0; a < FIRST; ++a)
      if (a < p.splits) sum = __builtin_fmaf(by[a], first[a], sum);
    int s = FIRST;
    for (; s + 8 <= p.splits; s += 8) {
      float x[8];
#pragma unroll
      for (int a = 0; a < 8; ++a) x[a] = in[(s + a) * width + d];
#pragma unroll
      for (int a = 0; a < 8; ++a) sum = __builtin_fmaf(by[s + a], x[a], sum);
    }
    for (; s < p.splits; ++s) sum = __builtin_fmaf(by[s], in[s * width + d], sum);
    o[d] = (T)(sum / weights);
  }
  if (head == 0 && d == 0) {
    p.length[slot] = seen < 0 ? 1 : seen + 1;
  }
}

struct CacheWriteParams {
  Series s;
  Rows k, v, kc, vc;
  int64_t kc_slot, vc_slot;
  int64_t *length;
  const int32_t *slots;
  int32_t n_slots, kv_heads, window, sinks, chunks;
};

constexpr int CW_ROWS = 32;

template <typename T> __device__ inline void copy8(T *to, const T *from, int d, int dim, bool vec) {
  if (d >= dim) return;
  if (vec) {
    *(Frag<T> *)(to + d) = *(const Frag<T> *)(from + d);
    return;
  }
  for (int e = d; e < d + 8 && e < dim; ++e) to[e] = from[e];
}

// A block takes CW_ROWS places of the cache of one series' slot and looks up which row belongs there.
template <typename T>
__global__ __launch_bounds__(256) void window_cache_write_kernel(CacheWriteParams p) {
  const int series = blockIdx.x / p.chunks, p0 = blockIdx.x % p.chunks * CW_ROWS;
  const int slot = slot_of(p.slots, series, p.n_slots);
  if (slot < 0) return;
  int64_t a = 0, b = p.s.n;
  if (p.s.offsets) { a = p.s.offsets[series]; b = p.s.offsets[series + 1]; }
  if (a < 0) a = 0;
  if (b > p.s.n) b = p.s.n;
  const int64_t m = b > a ? b - a : 0;
  const int cap = p.window + p.sinks;
  if (p0 == 0 && threadIdx.x == 0) p.length[slot] = m;
  for (int head = 0; head < p.kv_heads; ++head) {
    const T *kr = head_of<T>(p.k, head), *vr = head_of<T>(p.v, head);
    T *kc = (T *)p.kc.p + slot * p.kc_slot + head * p.kc.head, *vc = (T *)p.vc.p + slot * p.vc_slot + head * p.vc.head;
    const int pieces = TMP_MAX_HEAD_DIM / 8;
    for (int i = threadIdx.x; i < CW_ROWS * pieces; i += 256) {
      const int place = p0 + i / pieces, d = i % pieces * 8;
      if (place >= cap) break;
      int64_t t = place;
      if (place >= p.sinks) {
        if (m <= p.sinks) continue;
        int64_t back = (m - 1 - place) % p.window;  // rows since the last one that went to this place
        if (back < 0) back += p.window;
        t = m - 1 - back;
        if (t < p.sinks) continue;
      }
      if (t >= m) continue;
      copy8(kc + (int64_t)place * p.kc.row, kr + (a + t) * p.k.row, d, p.k.dim, p.k.vec && p.kc.vec);
      copy8(vc + (int64_t)place * p.vc.row, vr + (a + t) * p.v.row, d, p.v.dim, p.v.vec && p.vc.vec);
    }
  }
}

// ---- host ----------------------------------------------------------------------------------------

static bool cache_rows(const tmp_cache &c, int dim, int bytes, Rows *o) {
  const tmp_rows r = {c.p, c.row_stride, c.head_stride};
  const bool ok = rows_of(r, 2, dim, bytes, o);
  if (c.slot_stride % (16 / bytes)) o->vec = 0;
  return ok;
}
#define TMP_CACHE(what, ref, dim, bytes, to)                                                                   \
  TMP_REQUIRE(cache_rows(ref, dim, bytes, to), TMP_EUNSUPPORTED,                                               \
              "%s: the row stride of " #ref " must be at least its head size and below 2^22 elements, its pointer aligned", what)

static int step_check_common(int64_t n, int32_t n_slots, const int32_t *slots, int type, int heads, int dk, int dv,
                             const char *what) {
  TMP_REQUIRE(n >= 0 && n <= (1 << 24), TMP_EINVAL, "%s: row count must be in [0, 2^24]", what);
  // (every row looks through the slots of those before it)
  TMP_REQUIRE(!slots || n <= TMP_MAX_SLOT_ROWS, TMP_EUNSUPPORTED, "%s: at most %d rows with slots", what, TMP_MAX_SLOT_ROWS);
  TMP_REQUIRE(n_slots >= 0 && (slots || n <= n_slots), TMP_EINVAL, "%s: more rows than slots", what);
  TMP_REQUIRE(type == TMP_BF16 || type == TMP_F32, TMP_EUNSUPPORTED, "%s: type must be bfloat16 or float32", what);
  TMP_REQUIRE(heads > 0 && heads <= 65536, TMP_EINVAL, "%s: heads must be in [1, 65536]", what);
  TMP_REQUIRE(dk > 0 && dv > 0, TMP_EINVAL, "%s: head sizes must be positive", what);
  TMP_REQUIRE(dk <= TMP_MAX_HEAD_DIM && dv <= TMP_MAX_HEAD_DIM, TMP_EUNSUPPORTED, "%s: head sizes are limited to %d", what,
              TMP_MAX_HEAD_DIM);
  return TMP_OK;
}

static int window_step_check(const tmp_window_attention_step_args *a, const char *what) {
  TMP_REQUIRE(a != nullptr, TMP_EINVAL, "%s: null args", what);
  TMP_TRY(step_check_common(a->n, a->n_slots, a->slots, a->type, a->heads, a->dim_k, a->dim_v, what));
  TMP_REQUIRE(a->n * a->heads <= 2 * kMostBlocks, TMP_EUNSUPPORTED, "%s: too many rows x heads, at most 2^25 - 16", what);
  TMP_REQUIRE(a->kv_heads > 0 && a->heads % a->kv_heads == 0, TMP_EINVAL, "%s: heads must be a multiple of kv_heads", what);
  TMP_REQUIRE(a->window >= 1 && a->window < (1 << 30), TMP_EINVAL, "%s: window must be in [1, 2^30)", what);
  TMP_REQUIRE(a->sinks >= 0, TMP_EINVAL, "%s: sinks must be >= 0", what);
  TMP_REQUIRE(a->sinks <= TMP_MAX_SINKS, TMP_EUNSUPPORTED, "%s: at most %d sinks", what, TMP_MAX_SINKS);
  return TMP_OK;
}

// Rows of the cache that one wave takes: all of them once rows x heads give every compute unit eight
// waves (two a SIMD), else such a share that they do, 32 at least.  (Splits add at most WS_MOST_SPLITS waves to one for each
// row and head.)
static void window_step_split(const tmp_window_attention_step_args *a, int *splits, int *chunk) {
  const int64_t cap = (int64_t)a->window + a->sinks, group = a->heads / a->kv_heads;
  const int64_t units = (a->n > 0 ? a->n : 1) * a->kv_heads * ((group + 31) / 32);
  int64_t want = (WS_MOST_SPLITS + units - 1) / units;
  int64_t rows = (cap + want - 1) / want;
  rows = (rows + 31) / 32 * 32;
  *chunk = (int)rows;
  *splits = (int)((cap + rows - 1) / rows);
}

template <typename T, int D, bool VEC> static void window_step(const WindowStepParams &p, hipStream_t st) {
  const int group = p.heads / p.kv_heads;
  const int units = p.n * p.kv_heads * ((group + 31) / 32) * p.splits;
  {
    ProfScope ps("window_step_kernel", st);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(window_step_kernel<T, D, VEC>), dim3((units + 3) / 4), dim3(256), 4 * 32 * D * sizeof(T), st,
                       p, units);
  }
  ProfScope ps("window_join_kernel", st);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(window_join_kernel<T>), dim3(p.n * p.heads), dim3(128), 0, st, p);
}

}  // namespace tmp

using namespace tmp;

extern "C" int tmp_decay_attention_step(const tmp_decay_attention_step_args *a, void *stream) {
  clear_error();
  const char *what = "tmp_decay_attention_step";
  TMP_REQUIRE(a != nullptr, TMP_EINVAL, "%s: null args", what);
  TMP_TRY(step_check_common(a->n, a->n_slots, a->slots, a->type, a->heads, a->dim_k, a->dim_v, what));
  TMP_REQUIRE(a->n * a->heads <= kMostBlocks, TMP_EUNSUPPORTED, "%s: too many rows x heads, at most 2^24 - 8", what);
  TMP_REQUIRE(a->scale > 0.f && a->scale < INFINITY, TMP_EINVAL, "%s: scale must be positive and finite", what);
  if (a->n == 0) return TMP_OK;
  TMP_REQUIRE(a->q.p && a->k.p && a->v.p && a->out.p && a->log_decay && a->state, TMP_EINVAL, "%s: null pointer", what);
  const int b = a->type == TMP_F32 ? 4 : 2;
  DecayStepParams p;
  memset(&p, 0, sizeof(p));
  TMP_ROWS(what, a->q, a->n, a->dim_k, b, &p.q);
  TMP_ROWS(what, a->k, a->n, a->dim_k, b, &p.k);
  TMP_ROWS(what, a->v, a->n, a->dim_v, b, &p.v);
  TMP_ROWS(what, a->out, a->n, a->dim_v, b, &p.out);
  p.log_decay = a->log_decay; p.state = a->state; p.slots = a->slots;
  p.n = (int32_t)a->n; p.n_slots = a->n_slots; p.heads = a->heads; p.scale = a->scale;
  const bool vec = ((uintptr_t)a->state & 15) == 0 && a->dim_v % 4 == 0;
  const dim3 grid((unsigned)(a->n * a->heads)), block(256);
  hipStream_t st = (hipStream_t)stream;
  ProfScope ps("decay_step_kernel", st);
  if (a->type == TMP_F32) {
    if (vec) hipLaunchKernelGGL(HIP_KERNEL_NAME(decay_step_kernel<float, 4>), grid, block, 0, st, p);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(decay_step_kernel<float, 1>), grid, block, 0, st, p);
  } else {
    if (vec) hipLaunchKernelGGL(HIP_KERNEL_NAME(decay_step_kernel<__bf16, 4>), grid, block, 0, st, p);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(decay_step_kernel<__bf16, 1>), grid, block, 0, st, p);
  }
  TMP_CHECK_HIP(hipGetLastError());
  return TMP_OK;
}

extern "C" size_t tmp_window_attention_step_workspace_bytes(const tmp_window_attention_step_args *a) {
  if (!a || window_step_check(a, "tmp_window_attention_step") != TMP_OK) return 0;
  int splits, chunk;
  window_step_split(a, &splits, &chunk);
  return (size_t)(a->n > 0 ? a->n : 1) * a->heads * splits * (a->dim_v + 2) * 4;
}

extern "C" int tmp_window_attention_step(const tmp_window_attention_step_args *a, void *workspace, size_t workspace_bytes,
                                         void *stream) {
  clear_error();
  const char *what = "tmp_window_attention_step";
  TMP_TRY(window_step_check(a, what));
  TMP_REQUIRE(a->scale > 0.f && a->scale < INFINITY, TMP_EINVAL, "%s: scale must be positive and finite", what);
  if (a->n == 0) return TMP_OK;
  TMP_REQUIRE(a->q.p && a->k.p && a->v.p && a->out.p && a->k_cache.p && a->v_cache.p && a->length, TMP_EINVAL,
              "%s: null pointer", what);
  TMP_REQUIRE(workspace && workspace_bytes >= tmp_window_attention_step_workspace_bytes(a), TMP_EWORKSPACE,
              "%s: workspace too small", what);
  const int b = a->type == TMP_F32 ? 4 : 2;
  WindowStepParams p;
  memset(&p, 0, sizeof(p));
  TMP_ROWS(what, a->q, a->n, a->dim_k, b, &p.q);
  TMP_ROWS(what, a->k, a->n, a->dim_k, b, &p.k);
  TMP_ROWS(what, a->v, a->n, a->dim_v, b, &p.v);
  TMP_ROWS(what, a->out, a->n, a->dim_v, b, &p.out);
  TMP_CACHE(what, a->k_cache, a->dim_k, b, &p.kc);
  TMP_CACHE(what, a->v_cache, a->dim_v, b, &p.vc);
  p.kc_slot = a->k_cache.slot_stride; p.vc_slot = a->v_cache.slot_stride;
  p.length = a->length; p.slots = a->slots; p.part = (float *)workspace;
  p.n = (int32_t)a->n; p.n_slots = a->n_slots; p.heads = a->heads; p.kv_heads = a->kv_heads;
  p.window = a->window; p.sinks = a->sinks; p.scale = a->scale;
  window_step_split(a, &p.splits, &p.chunk);
  hipStream_t st = (hipStream_t)stream;
  const int d = padded_dim(a->dim_k > a->dim_v ? a->dim_k : a->dim_v);
  TMP_BY_FORM(window_step, a->type, d, p.kc.vec && p.vc.vec, p, st);
  TMP_CHECK_HIP(hipGetLastError());
  return TMP_OK;
}

extern "C" int tmp_window_cache_write(const tmp_window_cache_write_args *a, void *stream) {
  clear_error();
  const char *what = "tmp_window_cache_write";
  TMP_REQUIRE(a != nullptr, TMP_EINVAL, "%s: null args", what);
  TMP_REQUIRE(a->n >= 0 && a->n < (1ll << 31) - 65536, TMP_EINVAL, "%s: row count must be in [0, 2^31 - 65536)", what);
  TMP_SERIES(what, a);
  TMP_TRY(step_check_common(a->n_series, a->n_slots, a->slots, a->type, a->kv_heads, a->dim_k, a->dim_v, what));
  TMP_REQUIRE(a->window >= 1 && a->window < (1 << 30), TMP_EINVAL, "%s: window must be in [1, 2^30)", what);
  TMP_REQUIRE(a->sinks >= 0, TMP_EINVAL, "%s: sinks must be >= 0", what);
  TMP_REQUIRE(a->sinks <= TMP_MAX_SINKS, TMP_EUNSUPPORTED, "%s: at most %d sinks", what, TMP_MAX_SINKS);
  if (a->n_series == 0) return TMP_OK;
  TMP_REQUIRE(a->k_cache.p && a->v_cache.p && a->length && (a->n == 0 || (a->k.p && a->v.p)), TMP_EINVAL, "%s: null pointer", what);
  const int b = a->type == TMP_F32 ? 4 : 2;
  CacheWriteParams p;
  memset(&p, 0, sizeof(p));
  p.s.offsets = a->offsets; p.s.n_series = a->n_series; p.s.n = (int32_t)a->n;
  TMP_ROWS(what, a->k, a->n, a->dim_k, b, &p.k);
  TMP_ROWS(what, a->v, a->n, a->dim_v, b, &p.v);
  TMP_CACHE(what, a->k_cache, a->dim_k, b, &p.kc);
  TMP_CACHE(what, a->v_cache, a->dim_v, b, &p.vc);
  p.kc_slot = a->k_cache.slot_stride; p.vc_slot = a->v_cache.slot_stride;
  p.length = a->length; p.slots = a->slots; p.n_slots = a->n_slots; p.kv_heads = a->kv_heads;
  p.window = a->window; p.sinks = a->sinks;
  p.chunks = (p.window + p.sinks + CW_ROWS - 1) / CW_ROWS;
  TMP_REQUIRE((int64_t)p.chunks * a->n_series <= kMostBlocks, TMP_EUNSUPPORTED,
              "%s: too many series x rows of a cache, at most 2^24 - 8 times %d", what, CW_ROWS);
  const dim3 grid((unsigned)((int64_t)p.chunks * a->n_series)), block(256);
  hipStream_t st = (hipStream_t)stream;
  ProfScope ps("window_cache_write_kernel", st);
  if (a->type == TMP_F32) hipLaunchKernelGGL(HIP_KERNEL_NAME(window_cache_write_kernel<float>), grid, block, 0, st, p);
  else hipLaunchKernelGGL(HIP_KERNEL_NAME(window_cache_write_kernel<__bf16>), grid, block, 0, st, p);
  TMP_CHECK_HIP(hipGetLastError());
  return TMP_OK;
}
