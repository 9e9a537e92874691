// Operators on the distribution softmax(z / tau) over the vocabulary, from a [rows, V] block of logits (bf16 or fp32):
//
//   statistics  m = max z,  S = sum 2^t,  t = (z - m) c,  c = log2(e) / tau          (fp32, one pass, running maximum)
//               entropy H = ln S - ln 2 (sum 2^t t) / S
//               log-probability of a column i: (z_i - m) / tau - ln S
//               the k largest columns, equal logits in the order of their index
//   gradient    dz_i = 1/tau [ sum_j w_j (i = id_j) + q_i (alpha + beta ln q_i) ],  q_i = 2^(t_i - log2 S)
//               alpha = -sum_j w_j - g_H H,  beta = -g_H
//
// Log-probabilities (w = their upstream gradients) and distillation (w_j = -g mask tau^2 p_j, g_H = 0) share both
// kernels.  A row is kept as the pair (m, log2 S) and not as one log-sum-exp: with logits around 1000 the sum m + ln S
// would round off 3e-5 of every log-probability.
#include <algorithm>
#include <climits>
#include <type_traits>

#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"

namespace rk {

using bf16 = __nv_bfloat16;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// An exponent this low is zero in fp32; clamping there keeps 0 * t finite for columns at -inf.
constexpr float kMinExponent = -16384.f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// log2 of a row's sum.  The build's fast-math logarithm has an absolute error, which is everything when the sum is close to
// 1 (a confident prediction); this is s = 2^e f with f in [0.71, 1.42) and log f = 2 atanh u, u = (f - 1) / (f + 1), by
// atanh's power series: |u| < 0.172, the first term left out is below 2^-31 of the sum.
__device__ __forceinline__ float log2_row(float s) {
  if (!(s > 0.f && s < INFINITY)) return s == 0.f ? -INFINITY : s;
  const int e = (__float_as_int(s) - 0x3f3504f3) >> 23;
  const float f = __int_as_float(__float_as_int(s) - (e << 23));
  const float u = __fdiv_rn(f - 1.f, f + 1.f), v = u * u;
  float p = fmaf(v, 1.f / 11.f, 1.f / 9.f);
  p = fmaf(v, p, 1.f / 7.f);
  p = fmaf(v, p, 1.f / 5.f);
  p = fmaf(v, p, 1.f / 3.f);
  return fmaf(2.f * kLog2e * u, fmaf(v, p, 1.f), (float)e);
}

// A row seen as 16-byte units of the aligned addresses that hold it; the first and the last unit may be partly outside.
template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* x;
  int V, off, units;
  __device__ __forceinline__ Row(const T* p, int V_) : x(p), V(V_) {
    off = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    units = (V + off + E - 1) / E;
  }
  __device__ __forceinline__ int first(int u) const { return u * E - off; }
  __device__ __forceinline__ bool whole(int u) const { const int i = first(u); return i >= 0 && i + E <= V; }
  __device__ __forceinline__ void load(int u, float (&v)[E]) const {
    const int i0 = first(u);
    if (i0 >= 0 && i0 + E <= V) {
      const uint4 raw = *reinterpret_cast<const uint4*>(x + i0);
      unpack(raw, v);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = (i0 + e >= 0 && i0 + e < V) ? to_float(x[i0 + e]) : -INFINITY;
    }
  }
  static __device__ __forceinline__ void unpack(const uint4& raw, float (&v)[E]) {
    if constexpr (sizeof(T) == 2) {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
      for (int j = 0; j < 4; ++j) { const float2 f = __bfloat1622float2(h[j]); v[2 * j] = f.x; v[2 * j + 1] = f.y; }
    } else {
      const float* f = reinterpret_cast<const float*>(&raw);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = f[j];
    }
  }
};

// Integers in the order of the numbers (-0 and +0 equal, NaN below everything).
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0u;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

// Statistics relative to their own maximum: s1 = sum 2^t, s2 = sum 2^t t.
struct Stat { float m, s1, s2; };

__device__ __forceinline__ Stat merge(const Stat& a, const Stat& b, float c) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  const float da = a.m == -INFINITY ? 0.f : fmaxf((a.m - r.m) * c, kMinExponent);
  const float db = b.m == -INFINITY ? 0.f : fmaxf((b.m - r.m) * c, kMinExponent);
  const float fa = exp2_fast(da), fb = exp2_fast(db);
  r.s1 = fa * a.s1 + fb * b.s1;
  r.s2 = fa * (a.s2 + da * a.s1) + fb * (b.s2 + db * b.s1);
  return r;
}

__device__ __forceinline__ Stat shfl_xor(const Stat& a, int o) {
  return {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s1, o), __shfl_xor_sync(0xffffffffu, a.s2, o)};
}

constexpr int kThreads = 256;
constexpr int kUnroll = 4;
constexpr int kFewRowsThreads = 512, kManyRowsThreads = 128;     // of the forward kernel
constexpr int kCandidates = 512;
constexpr int kMaxTop = 64;
// The fast pass lifts columns below this to it (probability zero either way), so that 0 * t stays finite without a test of
// every exponent; a row whose maximum is that low itself is done again by the exact pass.
constexpr float kFloor = -1e30f;
// The fast pass keeps its reference until a logit exceeds it by this exponent (a thread then rescales once or twice a row):
// with the maximum itself as reference some lane of a warp would rescale in two of three units.
constexpr float kSlack = 8.f;

__device__ __forceinline__ uint32_t max_bf2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// One thread's statistics in the fast pass: t = z c - ref (one rounding, whatever the size of the logits), the sums in two
// halves, the largest logit and the first unit that holds it.
struct Running {
  float ref, limit, m, run_m;
  f2 s1, s2;
  int bu;
};

// A whole unit into the running statistics.
template <typename T, bool TOP>
__device__ __forceinline__ void take_fast(Running& st, uint4 raw, int u, float c, float slack) {
  f2 z[Row<T>::E / 2];
  float cm;
  if constexpr (sizeof(T) == 2) {
    const uint32_t low = 0xf149f149u;            // bf16 pair of about -1e30
    const uint32_t w[4] = {max_bf2(raw.x, low), max_bf2(raw.y, low), max_bf2(raw.z, low), max_bf2(raw.w, low)};
    const uint32_t mx = max_bf2(max_bf2(w[0], w[1]), max_bf2(w[2], w[3]));
    cm = fmaxf(__uint_as_float(mx << 16), __uint_as_float(mx & 0xffff0000u));
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = pack2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
  } else {
    const float w[4] = {max_nan(__uint_as_float(raw.x), kFloor), max_nan(__uint_as_float(raw.y), kFloor),
                        max_nan(__uint_as_float(raw.z), kFloor), max_nan(__uint_as_float(raw.w), kFloor)};
    cm = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
    z[0] = pack2(w[0], w[1]);
    z[1] = pack2(w[2], w[3]);
  }
  if (cm > st.limit) {
    const float ref = cm * c;
    // from no reference at all the sums are zero; a rise that overflows leaves a NaN, which the exact pass settles
    const float d = st.limit == -INFINITY ? 0.f : st.ref - ref, f = exp2_fast(d);
    const f2 ff = pack2(f, f);
    st.s2 = mul2(ff, fma2(pack2(d, d), st.s1, st.s2));
    st.s1 = mul2(ff, st.s1);
    st.ref = ref;
    st.limit = cm + slack;
  }
  if (TOP) { st.run_m = fmaxf(st.run_m, cm); if (cm > st.m) { st.m = cm; st.bu = u; } }
  else st.m = fmaxf(st.m, cm);
  const f2 nr = pack2(-st.ref, -st.ref), cc = pack2(c, c);
#pragma unroll
  for (int j = 0; j < Row<T>::E / 2; ++j) {
    const f2 t = fma2(z[j], cc, nr);
    float x, y;
    unpack2(t, x, y);
    const f2 p = pack2(exp2_fast(x), exp2_fast(y));
    st.s1 = add2(st.s1, p);
    st.s2 = fma2(p, t, st.s2);
  }
}

// Any unit, any values: columns at -inf, a row without a finite number, NaN.
template <typename T>
__device__ __forceinline__ void take_exact(Stat& st, int& bu, const float (&v)[Row<T>::E], int u, float c) {
  constexpr int E = Row<T>::E;
  float cm = v[0];
#pragma unroll
  for (int e = 1; e < E; ++e) cm = fmaxf(cm, v[e]);
  if (cm > st.m) {
    if (st.m != -INFINITY) {
      const float d = fmaxf((st.m - cm) * c, kMinExponent), f = exp2_fast(d);
      st.s2 = f * (st.s2 + d * st.s1);
      st.s1 *= f;
    }
    st.m = cm;
    bu = u;
  }
  if (st.m == -INFINITY) {
#pragma unroll
    for (int e = 0; e < E; ++e) if (v[e] != v[e]) st.s1 = v[e];
    return;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float t = (v[e] - st.m) * c;
    const float tc = t < kMinExponent ? kMinExponent : t;      // keeps a NaN
    const float p = exp2_fast(tc);
    st.s1 += p;
    st.s2 = fmaf(p, tc, st.s2);
  }
}

constexpr int kSub = 8;               // a thread's units in eight runs, each with its own maximum

template <int NT>
struct TopShared {
  int sel[NT], nsel, n, ntop, last, ngrp;
  int grp[kMaxTop * kSub];            // runs to look at again: thread and number of the run
  uint2 cand[kCandidates];
  uint2 top[kMaxTop];                 // the k largest in order: {value, column}
};

// The k largest columns of a row, into sh.top in order.  Thread t holds the units t, t + NT, ... and brings the key of its
// largest logit and the first unit that holds it.  The k-th largest of those keys bounds the k-th largest column from below,
// and of the threads above the bound the runs whose maximum reaches it are read again (`run` units of a thread each, from L2
// or memory): their elements above the bound are the candidates, ranked by counting.  Returns false, having chosen nothing,
// when the bound is not above `floor_key`.
template <typename T, int NT>
__device__ bool row_top(TopShared<NT>& sh, const float (&runs)[kSub][NT], const Row<T>& r, int run, int k, uint32_t key, int bu,
                        uint32_t floor_key) {
  constexpr int E = Row<T>::E;
  constexpr int SH = sizeof(T) == 2 ? 16 : 0;     // bf16 orders by the upper half of the key
  const int tid = threadIdx.x;
  const bool has = tid < r.units;
  key >>= SH;
  if (!has) key = 0u;                             // a thread without units has none
  // the largest bound that at least k thread maxima reach
  uint32_t bound = 0u;
  bool exact = false;
  for (int b = 31 - SH; b >= 0 && !exact; --b) {
    const uint32_t t = bound | (1u << b);
    const int n = __syncthreads_count(key >= t);
    if (n >= k) bound = t;
    exact = n == k;
  }
  if (exact) {
    // exactly the k largest, found before the last bit: the smallest of them is the tightest bound that they share
    const uint32_t mn = __reduce_min_sync(0xffffffffu, key >= bound ? key : 0xffffffffu);
    if ((tid & 31) == 0) sh.sel[tid >> 5] = (int)mn;
    __syncthreads();
    bound = 0xffffffffu;
    for (int w = 0; w < NT / 32; ++w) bound = min(bound, (uint32_t)sh.sel[w]);
    __syncthreads();
  }
  if (bound > 0u && bound <= (floor_key >> SH)) return false;
  if (tid == 0) { sh.nsel = 0; sh.n = 0; sh.ngrp = 0; }
  __syncthreads();
  int last = INT_MAX;                             // maxima equal to the bound count up to this unit
  if (!exact && bound > 0u) {
    // several threads share the bound: of those the ones with the lowest units, ranked by counting
    const int above = __syncthreads_count(key > bound);
    const bool tie = key == bound;
    if (tie) sh.sel[atomicAdd(&sh.n, 1)] = bu;
    if (tid == 0) sh.last = INT_MAX;
    __syncthreads();
    const int ties = sh.n;
    if (tie && ties > k - above) {
      int before = 0;
      for (int i = 0; i < ties; ++i) before += sh.sel[i] < bu;
      if (before == k - above - 1) sh.last = bu;
    }
    __syncthreads();
    last = sh.last;
    if (tid == 0) sh.n = 0;
    __syncthreads();
  }
  if (has && (key > bound || (key == bound && bu <= last))) sh.sel[atomicAdd(&sh.nsel, 1)] = tid;
  __syncthreads();
  const int nsel = sh.nsel;
  for (int i = tid; i < nsel * kSub; i += NT) {
    const int t = sh.sel[i / kSub];
    if ((order_key(runs[i % kSub][t]) >> SH) >= bound) sh.grp[atomicAdd(&sh.ngrp, 1)] = t * kSub + i % kSub;
  }
  __syncthreads();
  const int items = sh.ngrp * run;
  // every element of those runs, in any order
  auto each = [&](auto&& f) {
    for (int i = tid; i < items; i += NT) {
      const int g = sh.grp[i / run], u = g / kSub + ((g % kSub) * run + i % run) * NT;
      if (u >= r.units) continue;
      float v[E];
      r.load(u, v);
      const int i0 = r.first(u);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int idx = i0 + e;
        if (idx >= 0 && idx < r.V && v[e] == v[e]) f(order_key(v[e]) >> SH, idx, u, v[e]);
      }
    }
  };
  auto total = [&](int mine) {                    // sum over the CTA
    if (tid == 0) sh.n = 0;
    __syncthreads();
    atomicAdd(&sh.n, mine);
    __syncthreads();
    const int n = sh.n;
    __syncthreads();
    return n;
  };
  auto push = [&](float v, int idx) {
    const int at = atomicAdd(&sh.n, 1);
    if (at < kCandidates) sh.cand[at] = make_uint2(__float_as_uint(v), (uint32_t)idx);
  };
  each([&](uint32_t kk, int idx, int u, float v) { if (kk > bound || (kk == bound && u <= last)) push(v, idx); });
  __syncthreads();
  int n = sh.n;
  __syncthreads();
  if (n > kCandidates) {
    // the chosen threads hold long runs above the bound (sorted or blockwise rows): the exact k-th of their elements, by
    // bisection over the value and then over the index
    uint32_t kth = 0u;
    for (int b = 31 - SH; b >= 0; --b) {
      const uint32_t t = kth | (1u << b);
      int cnt = 0;
      each([&](uint32_t kk, int, int, float) { cnt += kk >= t; });
      if (total(cnt) >= k) kth = t;
    }
    int gt = 0;
    each([&](uint32_t kk, int, int, float) { gt += kk > kth; });
    const int need = k - total(gt);
    int lim = 0;                                  // elements equal to the k-th count up to this index
    for (int b = 30; b >= 0; --b) {
      int cnt = 0;
      each([&](uint32_t kk, int idx, int, float) { cnt += kk == kth && idx < (lim | (1 << b)); });
      if (total(cnt) < need) lim |= 1 << b;
    }
    if (tid == 0) sh.n = 0;
    __syncthreads();
    each([&](uint32_t kk, int idx, int, float v) { if (kk > kth || (kk == kth && idx <= lim)) push(v, idx); });
    __syncthreads();
    n = min(sh.n, kCandidates);
  }
  for (int i = tid; i < n; i += NT) {
    const uint2 mine = sh.cand[i];
    const float v = __uint_as_float(mine.x);
    int rank = 0;
    for (int j = 0; j < n; ++j) {
      const float w = __uint_as_float(sh.cand[j].x);
      rank += w > v || (w == v && sh.cand[j].y < mine.y);
    }
    if (rank < k) sh.top[rank] = mine;
  }
  if (tid == 0) sh.ntop = min(n, k);
  __syncthreads();
  return true;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// How far a thread of the forward kernel reads ahead (kStages batches of kBatch units), and how many CTAs share an SM.
template <int NT, bool TOP> struct Ahead { static constexpr int kBatch = 2, kStages = TOP ? 4 : 5, kResident = 1280 / NT; };
template <bool TOP> struct Ahead<kFewRowsThreads, TOP> { static constexpr int kBatch = 1, kStages = TOP ? 3 : 4, kResident = 2; };

// Forward: one CTA per row, its threads over the row's 16-byte units.  A thread copies its own units into its own places of
// shared memory, several batches ahead, so that no thread waits for another and the copies in flight cost no registers.
// Bound by memory: 4096 x 65536 bf16 take 85.7 us, 6.27 TB/s (as fp32, 4096 x 32768, 82.4 us; a plain read 75.6 us).  With two
// register buffers of four units instead of the ring it was 106 us; one CTA going from row to row and reading ahead into the
// next one 113 us, for the registers that costs.
// kDo says what else a row is for: nothing, its alternatives, or its distillation loss.
enum RowDo { kOnlyStats, kAlternatives, kDistill };
template <typename T, RowDo kDo, int NT>
__global__ void __launch_bounds__(NT, Ahead<NT, kDo == kAlternatives>::kResident) row_stats_kernel(RowStatsArgs a) {
  constexpr bool TOP = kDo == kAlternatives;
  constexpr int E = Row<T>::E;
  constexpr int W = NT / 32;
  constexpr int kBatch = Ahead<NT, TOP>::kBatch, kStages = Ahead<NT, TOP>::kStages;
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float c = kLog2e * a.inv_tau;
  if (kDo == kDistill && a.mask != nullptr && a.mask[row] == 0.f) {
    // a row that does not count is not read: whatever it holds stays out of the sums
    if (tid == 0) {
      a.stats[row] = make_float2(0.f, 0.f);
      a.row_loss[row] = 0.f;
    }
    return;
  }
  __shared__ float sm_m[W];
  __shared__ float2 sm_s[W], sm_l[W];
  __shared__ float sm_ln;
  __shared__ __align__(128) uint4 ring[kStages * kBatch][NT];     // on whole lines: 48 bytes off cost 6 us of 90
  using Top = typename std::conditional<TOP, TopShared<NT>, int>::type;
  static_assert(sizeof(Top) <= sizeof(ring), "the alternatives are chosen when the ring has been read");
  Top& sh = *reinterpret_cast<Top*>(&ring[0][0]);
  __shared__ float runs[TOP ? kSub : 1][NT];          // the maximum of each run of a thread's units
  const Row<T> r(reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld, a.V);

  auto block_max = [&](float m) {
    m = warp_max(m);
    if (lane == 0) sm_m[warp] = m;
    __syncthreads();
    m = sm_m[0];
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, sm_m[w]);
    return m;
  };
  auto block_sum2 = [&](float2 (&sm)[W], float x, float y) {
    x = warp_sum(x);
    y = warp_sum(y);
    if (lane == 0) sm[warp] = make_float2(x, y);
    __syncthreads();
    float2 t = sm[0];
#pragma unroll
    for (int w = 1; w < W; ++w) { t.x += sm[w].x; t.y += sm[w].y; }
    return t;
  };
  // whole units are [b0, b1); the row's first and last unit may be partly outside of it
  const int b0 = r.whole(0) ? 0 : 1, b1 = r.whole(r.units - 1) ? r.units : r.units - 1;
  const uint4* base = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(r.x) & ~uintptr_t(15)) + tid;
  const uint32_t mine = smem_u32(&ring[0][tid]);
  const int nb = (r.units + kBatch * NT - 1) / (kBatch * NT), run = (nb + kSub - 1) / kSub;   // batches; batches in a run
  // the teacher's alternatives of a distillation: this thread's probabilities and columns
  constexpr int kMine = (256 + NT - 1) / NT;
  float t_p[kMine], t_plogp = 0.f;
  int t_col[kMine];
  auto issue = [&](int blk, int stage) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int at = (blk * kBatch + i) * NT;
      if (at + tid >= b0 && at + tid < b1) cp_async16(mine + (uint32_t)((stage * kBatch + i) * NT * 16), base + at);
    }
    cp_async_commit();                                // past the row's end an empty group
  };
#pragma unroll
  for (int j = 0; j < kStages; ++j) issue(j, j);
  // what the row's end needs of single columns is asked for now: there, two loads in a row would be the CTA's whole work
  int id = -1;
  float z_id = 0.f;
  if (tid == 0 && a.logprob != nullptr) {
    id = a.ids[row];
    if (id >= 0 && id < a.V) z_id = to_float(r.x[id]);
  }
  float z_t[kMine];
  if constexpr (kDo == kDistill) {                    // while the first units are on their way
    float x[kMine], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int j = tid + i * NT;
      const size_t at = (size_t)row * a.K + j;
      t_col[i] = j < a.K ? a.t_ids[at] : -1;
      x[i] = -INFINITY;
      if (t_col[i] >= 0 && t_col[i] < a.V)
        x[i] = a.t_bf16 ? to_float(static_cast<const bf16*>(a.t_logits)[at]) : static_cast<const float*>(a.t_logits)[at];
      m = fmaxf(m, x[i]);                             // absent: outside of the vocabulary, -inf or NaN
    }
    m = block_max(m);
    float s = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const float t = fmaxf((x[i] - m) * c, kMinExponent);
      t_p[i] = x[i] > -INFINITY ? exp2_fast(t) : 0.f;
      s += t_p[i];
      s2 = fmaf(t_p[i], t, s2);
    }
    const float2 t = block_sum2(sm_l, s, s2);
    const float inv = t.x > 0.f ? 1.f / t.x : 0.f;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      t_p[i] *= inv;
      z_t[i] = t_p[i] > 0.f ? to_float(r.x[t_col[i]]) : 0.f;
      if (tid + i * NT < a.K) a.t_prob[(size_t)row * a.K + tid + i * NT] = t_p[i];
    }
    t_plogp = t.x > 0.f ? kLn2 * (t.y * inv - log2_row(t.x)) : INFINITY;       // sum p ln p; infinite without alternatives
    __syncthreads();                                  // sm_m and sm_l are written again below
  }
  Running st{0.f, -INFINITY, -INFINITY, -INFINITY, 0ull, 0ull, tid};
  const float slack = kSlack / c;
  // lifted to the floor, the columns outside of the row have no part
  auto ragged = [&](int u) {
    float v[E];
    r.load(u, v);
    uint4 raw;
    if constexpr (sizeof(T) == 2) {
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
    } else {
      raw = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    take_fast<T, TOP>(st, raw, u, c, slack);
  };
  if (b0 == 1 && tid == 0) ragged(0);
  int stage = 0, in_run = 0, which = 0, j = 0;
  // one batch; `inside`: it and the one requested in its place are whole units for every thread
  auto step = [&](auto inside) {
    cp_async_wait<kStages - 1>();
    uint4 raw[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) raw[i] = ring[stage * kBatch + i][tid];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int u = (j * kBatch + i) * NT + tid;
      if (inside || (u >= b0 && u < b1)) take_fast<T, TOP>(st, raw[i], u, c, slack);
    }
    if (inside) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        cp_async16(mine + (uint32_t)((stage * kBatch + i) * NT * 16), base + ((j + kStages) * kBatch + i) * NT);
      cp_async_commit();
    } else {
      issue(j + kStages, stage);
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;
    ++j;
    if (TOP && (++in_run == run || j == nb)) {
      runs[which++][tid] = st.run_m;
      st.run_m = -INFINITY;
      in_run = 0;
    }
  };
  const int inner = b1 / (kBatch * NT) - kStages;     // batches with kStages full ones behind them
  if (b0 == 1 && inner > 0) step(std::false_type());
  while (j < inner) step(std::true_type());
  while (j < nb) step(std::false_type());
  cp_async_wait<0>();
  if (b1 < r.units && r.units - 1 >= b0 && tid == (r.units - 1) % NT) {
    ragged(r.units - 1);
    if (TOP) runs[which - 1][tid] = fmaxf(runs[which - 1][tid], st.run_m);      // it lies in the last batch
  }

  float m = block_max(st.m);
  float x0, x1, y0, y1;
  unpack2(st.s1, x0, x1);
  unpack2(st.s2, y0, y1);
  // from the thread's reference to the row's maximum
  const float d = st.limit == -INFINITY ? 0.f : fmaf(-m, c, st.ref), f = exp2_fast(d), s1 = x0 + x1;
  float2 tot = block_sum2(sm_s, f * s1, f * fmaf(d, s1, y0 + y1));
  // overflow, -inf times zero, NaN, a row at the floor: the exact pass below
  bool done = m > 0.1f * kFloor && fabsf(tot.x) < INFINITY && fabsf(tot.y) < INFINITY;
  if constexpr (TOP) {
    if (done) done = row_top<T, NT>(sh, runs, r, run * kBatch, a.top_k, order_key(st.m), st.bu, order_key(kFloor * 0.99f));
  }
  if (!done) {
    Stat se{-INFINITY, 0.f, 0.f};
    int bu = tid;
    for (int u = tid; u < r.units; u += NT) { float v[E]; r.load(u, v); take_exact<T>(se, bu, v, u, c); }
    __syncthreads();
    m = block_max(se.m);
    const float de = se.m == -INFINITY ? 0.f : fmaxf((se.m - m) * c, kMinExponent), fe = exp2_fast(de);
    tot = block_sum2(sm_s, fe * se.s1, fe * fmaf(de, se.s1, se.s2));
    if constexpr (TOP) {
      for (int i = 0; i < kSub; ++i) runs[i][tid] = INFINITY;          // every run of a chosen thread
      __syncthreads();
      row_top<T, NT>(sh, runs, r, run * kBatch, a.top_k, order_key(se.m), bu, 0u);
    }
  }
  if (tid == 0) {
    const float l2s = log2_row(tot.x);                // -inf for a row without a number, NaN for a row with one
    const float ln_s = tot.x > 0.f ? l2s * kLn2 : __int_as_float(0x7fffffff);
    a.stats[row] = make_float2(m, l2s);
    if (a.entropy != nullptr) a.entropy[row] = tot.x > 0.f ? ln_s - kLn2 * (tot.y / tot.x) : ln_s;
    // an id outside the vocabulary is no token: nothing to score
    if (a.logprob != nullptr) a.logprob[row] = id >= 0 && id < a.V ? (z_id - m) * a.inv_tau - ln_s : 0.f;
    sm_ln = ln_s;
  }
  if constexpr (kDo == kDistill) {
    // mask tau^2 (sum p ln p - sum p ln q) over the teacher's alternatives
    float acc = 0.f, psum = 0.f;
#pragma unroll
    for (int i = 0; i < kMine; ++i)
      if (t_p[i] > 0.f) { acc += t_p[i] * ((z_t[i] - m) * a.inv_tau); psum += t_p[i]; }
    const float2 t = block_sum2(sm_l, acc, psum);
    if (tid == 0)
      a.row_loss[row] = t_plogp < INFINITY ? (a.mask != nullptr ? a.mask[row] : 1.f) * a.tau * a.tau * (t_plogp - (t.x - t.y * sm_ln)) : 0.f;
  }
  if constexpr (TOP) {
    __syncthreads();
    for (int i = tid; i < a.top_k; i += NT) {
      const bool there = i < sh.ntop;                 // fewer than k numbers in the row: -1, NaN
      a.top_ids[(size_t)row * a.top_k + i] = there ? (int)sh.top[i].y : -1;
      a.top_logprobs[(size_t)row * a.top_k + i] =
          there ? (__uint_as_float(sh.top[i].x) - m) * a.inv_tau - sm_ln : __int_as_float(0x7fffffff);
    }
  }
}

// Backward: a CTA takes `iters` blocks of kThreads * kUnroll units of a row, the next block's logits in flight while one is
// written.  Dense part first, then the columns of the sparse list that lie in this CTA's part are written again with their
// whole value (the list may name a column more than once).  Rows go from the last to the first: behind a forward pass the
// end of the logits is what L2 still holds.  Bound by memory: 4096 x 65536 bf16 take 163 us behind the forward pass, 6.6 TB/s
// of reading and writing, the rate of a plain copy.
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(kThreads, 4) row_grad_kernel(RowGradArgs a, int iters) {
  constexpr int E = Row<T>::E;
  constexpr int B0 = kThreads * kUnroll;
  const int row = a.rows - 1 - (int)blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld;
  T* out = reinterpret_cast<T*>(a.dlogits) + (size_t)row * a.ldd;
  const Row<T> o(out, a.V);                           // units by the output's alignment
  const int u0 = blockIdx.x * B0 * iters, u1 = min(o.units, u0 + B0 * iters);
  if (u0 >= u1) return;
  const bool congruent = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  auto fetch = [&](uint4 (&buf)[kUnroll], int u) {
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int ui = u + i * kThreads;
      if (congruent && ui < u1 && o.whole(ui)) buf[i] = __ldg(reinterpret_cast<const uint4*>(x + o.first(ui)));
    }
  };
  // the logits are requested before anything else, so that the row's scalars arrive in their shadow
  uint4 cur[kUnroll];
  fetch(cur, u0 + tid);
  float scale = a.weight_mul;
  if (a.g_scale != nullptr) scale *= a.g_scale[0];
  if (a.mask != nullptr) scale = a.mask[row] == 0.f ? 0.f : scale * a.mask[row];
  const float g_h = ENTROPY ? a.g_entropy[row] : 0.f;
  const float2 st = a.stats[row];
  __shared__ float sm_w[kThreads / 32];
  float wsum = 0.f;
  int any = g_h != 0.f;
  if (scale != 0.f)
    for (int j = tid; j < a.K; j += kThreads) {
      const int id = a.ids[(size_t)row * a.K + j];
      const float w = a.w[(size_t)row * a.K + j];
      if (id >= 0 && id < a.V && w != 0.f) { wsum += w; any = 1; }
    }
  wsum = warp_sum(wsum);
  if (lane == 0) sm_w[warp] = wsum;
  any = __syncthreads_or(any);
  wsum = 0.f;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) wsum += sm_w[w];
  const float c = kLog2e * a.inv_tau;
  const float m = st.x, l2s = st.y;
  const float A = a.inv_tau * (-scale * wsum - (ENTROPY && g_h != 0.f ? g_h * a.entropy[row] : 0.f));
  const float B = -g_h * a.inv_tau * kLn2;            // times log2 q
  const f2 nm = pack2(-m, -m), cc = pack2(c, c), nl = pack2(-l2s, -l2s), A2 = pack2(A, A), B2 = pack2(B, B);
  auto value2 = [&](float& z0, float& z1) {
    f2 t = fma2(add2(pack2(z0, z1), nm), cc, nl);
    float t0, t1;
    unpack2(t, t0, t1);
    if (ENTROPY) {                                    // a column at -inf: 0 * B t
      t0 = t0 < kMinExponent ? kMinExponent : t0;
      t1 = t1 < kMinExponent ? kMinExponent : t1;
      t = pack2(t0, t1);
    }
    const f2 q = pack2(exp2_fast(t0), exp2_fast(t1));
    unpack2(mul2(q, ENTROPY ? fma2(B2, t, A2) : A2), z0, z1);
  };
  for (int ub = u0; ub < u1; ub += B0) {
    uint4 nxt[kUnroll];
    fetch(nxt, ub + B0 + tid);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int u = ub + tid + i * kThreads;
      if (u >= u1) break;
      const int i0 = o.first(u);
      const bool whole = o.whole(u);
      float v[E];
      if (!any) {
        // nothing flows into this row (padding, a masked row): its logits are not used, so they may hold anything
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = 0.f;
      } else {
        if (congruent && whole) Row<T>::unpack(cur[i], v);
        else {
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] = (i0 + e >= 0 && i0 + e < a.V) ? to_float(x[i0 + e]) : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < E; e += 2) value2(v[e], v[e + 1]);
      }
      if (whole) {
        uint4 w;
        if constexpr (sizeof(T) == 2) {
          __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
          for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        } else {
          w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        }
        *reinterpret_cast<uint4*>(out + i0) = w;
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) if (i0 + e >= 0 && i0 + e < a.V) out[i0 + e] = from_float<T>(v[e]);
      }
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) cur[i] = nxt[i];
  }
  if (!any) return;
  __syncthreads();
  const int lo = o.first(u0), hi = o.first(u1);
  for (int j = tid; j < a.K; j += kThreads) {
    const int id = a.ids[(size_t)row * a.K + j];
    if (id < 0 || id >= a.V || id < lo || id >= hi) continue;
    float w = 0.f;
    for (int i = 0; i < a.K; ++i) if (a.ids[(size_t)row * a.K + i] == id) w += a.w[(size_t)row * a.K + i];
    float d = to_float(x[id]), unused = d;
    value2(d, unused);
    out[id] = from_float<T>(d + scale * w * a.inv_tau);
  }
}

// A teacher's alternatives, one warp per row: p = softmax of their logits / tau over those that are there (id inside the
// vocabulary, logit above -inf), sorted by id so that a pass over the columns in order meets them in order; absent ones
// go last with the id INT_MAX and p = 0.  Also sum p ln p, whether the row has any, and where its ids enter each block of 256
// columns (a search by the product's epilogue: 65 us against 60 at 512 x 768 x 65536 with 16 alternatives, 77 against 66 with 128).
template <typename T>
__global__ void __launch_bounds__(256) teacher_prepare_kernel(const int* __restrict__ ids, const T* __restrict__ logits,
                                                              int rows, int K, int V, float inv_tau, int* __restrict__ out_ids,
                                                              float* __restrict__ out_p, float2* __restrict__ out_row,
                                                              uint16_t* __restrict__ first) {
  extern __shared__ int sm_ids[];                     // [8][2][K]: as given, in order
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x * 8 + warp;
  if (row >= rows) return;
  int* my = sm_ids + warp * 2 * K;
  const int* rid = ids + (size_t)row * K;
  const T* rl = logits + (size_t)row * K;
  float m = -INFINITY;
  for (int j = lane; j < K; j += 32) {
    int id = rid[j];
    const float x = to_float(rl[j]);
    if (id < 0 || id >= V || !(x > -INFINITY)) id = INT_MAX;
    else m = fmaxf(m, x);
    my[j] = id;
  }
  m = warp_max(m);
  __syncwarp();
  const float c = kLog2e * inv_tau;
  float s = 0.f, s2 = 0.f;
  for (int j = lane; j < K; j += 32)
    if (my[j] != INT_MAX) {
      const float t = fmaxf((to_float(rl[j]) - m) * c, kMinExponent), e = exp2_fast(t);
      s += e;
      s2 = fmaf(e, t, s2);
    }
  s = warp_sum(s);
  s2 = warp_sum(s2);
  const float inv = s > 0.f ? 1.f / s : 0.f;
  for (int j = lane; j < K; j += 32) {
    const int id = my[j];
    int rank = 0;
    for (int i = 0; i < K; ++i) rank += my[i] < id || (my[i] == id && i < j);
    my[K + rank] = id;
    out_ids[(size_t)row * K + rank] = id;
    out_p[(size_t)row * K + rank] = id != INT_MAX ? exp2_fast(fmaxf((to_float(rl[j]) - m) * c, kMinExponent)) * inv : 0.f;
  }
  if (lane == 0) out_row[row] = s > 0.f ? make_float2(kLn2 * (s2 * inv - log2_row(s)), 1.f) : make_float2(0.f, 0.f);
  __syncwarp();
  const int blocks = (V + 255) / 256;
  for (int t = lane; t < blocks; t += 32) {
    int lo = 0, hi = K;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (my[K + mid] < t * 256) lo = mid + 1; else hi = mid;
    }
    first[(size_t)row * blocks + t] = (uint16_t)lo;
  }
}

// Totals of row vectors, one CTA each: a fixed order, sums in 64 bits.
__global__ void __launch_bounds__(1024) row_totals_kernel(RowTotalsArgs a) {
  __shared__ double sm[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float* in = a.in[blockIdx.x];
  double s = 0.0;
  if (in == nullptr) s = threadIdx.x == 0 ? (double)a.rows : 0.0;
  else for (int r = threadIdx.x; r < a.rows; r += 1024) s += (double)in[r];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) sm[warp] = s;
  __syncthreads();
  if (warp == 0) {
    s = sm[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) *a.out[blockIdx.x] = (float)s;
  }
}

// ---- through the head: folding the tiles of the product's epilogue (one warp per row) -------------------------------------

__global__ void __launch_bounds__(256) head_prob_combine_kernel(const float4* __restrict__ tiles, int ntiles,
                                                                const int* __restrict__ target, const float* __restrict__ target_z,
                                                                int rows, int V, float inv_tau, float* __restrict__ logprob,
                                                                float* __restrict__ entropy, float4* __restrict__ stat) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= rows) return;
  const float c = kLog2e * inv_tau;
  Stat st{-INFINITY, 0.f, 0.f};
  for (int t = lane; t < ntiles; t += 32) {
    const float4 v = tiles[(size_t)row * ntiles + t];
    st = merge(st, Stat{v.x, v.y, v.z}, c);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) st = merge(st, shfl_xor(st, o), c);
  if (lane == 0) {
    const float l2s = log2_row(st.s1), ln_s = st.s1 > 0.f ? l2s * kLn2 : __int_as_float(0x7fffffff);
    const float h = ln_s - kLn2 * (st.s2 / st.s1);
    const int id = target[row];
    logprob[row] = id >= 0 && id < V ? (target_z[row] - st.m) * inv_tau - ln_s : 0.f;
    entropy[row] = h;
    stat[row] = make_float4(st.m, 0.f, l2s, h);
  }
}

__global__ void __launch_bounds__(256) head_distill_combine_kernel(const float4* __restrict__ tiles, int ntiles, HeadDistillRows a) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= a.rows) return;
  const float inv_tau = 1.f / a.tau, c = kLog2e * inv_tau;
  float m = -INFINITY, s = 0.f, st = 0.f;             // sums at temperature 1 and at tau
  int am = INT_MAX;
  auto fold = [&](float m2, float s2, float st2, int am2) {
    const float mm = fmaxf(m, m2);
    const float d1 = m == -INFINITY ? 0.f : m - mm, d2 = m2 == -INFINITY ? 0.f : m2 - mm;
    s = s * exp2_fast(d1 * kLog2e) + s2 * exp2_fast(d2 * kLog2e);
    st = st * exp2_fast(d1 * c) + st2 * exp2_fast(d2 * c);
    am = m2 > m || (m2 == m && am2 < am) ? am2 : am;
    m = mm;
  };
  for (int t = lane; t < ntiles; t += 32) {
    const float4 v = tiles[(size_t)row * ntiles + t];
    fold(v.x, v.y, v.z, __float_as_int(v.w));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    fold(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o), __shfl_xor_sync(0xffffffffu, st, o),
         __shfl_xor_sync(0xffffffffu, am, o));
  const float l2s1 = log2_row(s), l2st = log2_row(st);
  float acc = 0.f;
  for (int j = lane; j < a.K; j += 32) {
    const float p = a.t_prob[(size_t)row * a.K + j];
    if (p > 0.f) acc += p * ((a.cols_z[(size_t)row * a.K + j] - m) * inv_tau - l2st * kLn2);
  }
  acc = warp_sum(acc);
  if (lane == 0) {
    const float w = a.mask != nullptr ? a.mask[row] : 1.f;
    const float2 tr = a.t_row[row];
    const int tgt = a.target[row];
    const float w_ce = tgt >= 0 && tgt < a.V ? w : 0.f, w_kd = tr.y > 0.f ? w : 0.f;
    a.ce[row] = w_ce != 0.f ? w_ce * (l2s1 * kLn2 - (a.target_z[row] - m)) : 0.f;
    a.kd[row] = w_kd != 0.f ? w_kd * a.tau * a.tau * (tr.x - acc) : 0.f;
    a.l2[row] = 0.5e-4f * m * m;
    a.ce_count[row] = w_ce;
    a.stat[row] = make_float4(m, l2s1, l2st, 0.f);
    a.weight[row] = make_float2(w_ce, w_kd);
    a.argmax[row] = am;
  }
}

// The gradient of one logit of a row, dense part.
struct HeadCoef {
  float m, c, l2s1, l2st, A, B, g_ce, g_kd, unit;
  __device__ __forceinline__ float prob(float z) const {
    const float l = fmaf(z - m, c, -l2st);
    return exp2_fast(l) * fmaf(B, l, A);
  }
  __device__ __forceinline__ float distill(float z) const {
    const float d = z - m;
    return fmaf(g_kd, exp2_fast(fmaf(d, c, -l2st)), g_ce * exp2_fast(fmaf(d, kLog2e, -l2s1)));
  }
};

// What flows into a row.  `live` is false where nothing does: such a row gets zeros, whatever its logits.
template <bool DISTILL>
__device__ __forceinline__ HeadCoef head_coef(const HeadFix& a, int row, float& gl, bool& live) {
  const float inv_tau = 1.f / a.tau;
  const float4 s = a.stat[row];
  HeadCoef k{s.x, kLog2e * inv_tau, s.y, s.z, 0.f, 0.f, 0.f, 0.f, 1.f};
  gl = 0.f;
  if (DISTILL) {
    const float2 w = a.weight[row];
    k.unit = head_unit(a.g0, a.g1, a.tau);
    k.g_ce = a.g0 != nullptr ? __fdiv_rn(a.g0[0], k.unit) * w.x : 0.f;
    k.g_kd = a.g1 != nullptr ? __fdiv_rn(a.g1[0] * a.tau, k.unit) * w.y : 0.f;
    live = k.g_ce != 0.f || k.g_kd != 0.f;
  } else {
    const int id = a.target[row];
    gl = a.g0 != nullptr && id >= 0 && id < a.V ? a.g0[row] : 0.f;
    const float gh = a.g1 != nullptr ? a.g1[row] : 0.f;
    k.A = inv_tau * (-gl - (gh != 0.f ? gh * s.w : 0.f));
    k.B = -gh * inv_tau * kLn2;
    gl *= inv_tau;
    live = gl != 0.f || gh != 0.f;
  }
  return k;
}

// The listed columns of a row within [lo, hi), by `n` threads of which this is number t: dense part and one-hot terms.
__device__ __forceinline__ void prob_listed(const HeadFix& a, const HeadCoef& k, float gl, int row, int lo, int hi) {
  const int id = a.target[row];
  if (gl != 0.f && id >= lo && id < hi)
    reinterpret_cast<bf16*>(a.dz)[(size_t)row * a.ld + id] = f2bf(k.prob(a.target_z[row]) + gl);
}
__device__ __forceinline__ void distill_listed(const HeadFix& a, const HeadCoef& k, int row, int lo, int hi, int t, int n) {
  const int tgt = k.g_ce != 0.f ? a.target[row] : -1, am = a.argmax[row];
  const float g_l2 = a.g_l2 != nullptr ? __fdiv_rn(a.g_l2[0], k.unit) * 1e-4f * k.m : 0.f;
  const int* ids = a.t_ids + (size_t)row * a.K;
  bf16* dz = reinterpret_cast<bf16*>(a.dz) + (size_t)row * a.ld;
  auto put = [&](int col, float z, float p) {
    float d = 0.f;
    if (k.g_kd != 0.f) d = k.g_kd * (exp2_fast(fmaf(z - k.m, k.c, -k.l2st)) - p);
    if (k.g_ce != 0.f) d += k.g_ce * (exp2_fast(fmaf(z - k.m, kLog2e, -k.l2s1)) - (col == tgt ? 1.f : 0.f));
    if (col == am) d += g_l2;
    dz[col] = f2bf(d);
  };
  auto listed = [&](int col) {                        // the ids are in order
    int l = 0, h = a.K;
    while (l < h) { const int mid = (l + h) >> 1; if (ids[mid] < col) l = mid + 1; else h = mid; }
    return l < a.K && ids[l] == col;
  };
  for (int j = t; j < a.K; j += n) {
    const int id = ids[j];
    if (id < lo || id >= hi || (j > 0 && ids[j - 1] == id)) continue;      // absent ones are INT_MAX; the first of a run writes
    float p = 0.f;
    for (int i = j; i < a.K && ids[i] == id; ++i) p += a.t_prob[(size_t)row * a.K + i];
    put(id, a.cols_z[(size_t)row * a.K + j], p);
  }
  if (t == 0 && tgt >= lo && tgt < hi && !listed(tgt)) put(tgt, a.target_z[row], 0.f);
  if (t == n - 1 && am >= lo && am < hi && am != tgt && !listed(am)) put(am, k.m, 0.f);
}

__global__ void __launch_bounds__(256) head_prob_fix_kernel(HeadFix a) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= a.rows) return;
  float gl;
  bool live;
  const HeadCoef k = head_coef<false>(a, row, gl, live);
  prob_listed(a, k, gl, row, 0, a.V);
}

// One warp per row.
__global__ void __launch_bounds__(256) head_distill_fix_kernel(HeadFix a) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  float gl;
  bool live;
  const HeadCoef k = head_coef<true>(a, row, gl, live);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.unit = k.unit;
  distill_listed(a, k, row, 0, a.V, threadIdx.x & 31, 32);
}

// Gradient from kept logits: fp16 distances in, bf16 out.  A thread takes 8 columns at a time (16 bytes in, 16 out), a CTA
// `iters` blocks of 8192 columns, the next block's in flight while one is written.  Rows from the last to the first, as above.
// Bound by memory and, with two temperatures, by two exponentials an element: 16384 x 65536 take 811 us, 5.3 TB/s; 4093 x
// 65536 with one 170 us, 6.3 TB/s.
template <bool DISTILL>
__global__ void __launch_bounds__(256, 4) head_grad_kept_kernel(HeadFix a, const __half* __restrict__ z, int64_t ldz,
                                                                const float* __restrict__ z_top, int iters) {
  constexpr int kEach = 4, kBlock = 256 * 8 * kEach;
  const int row = a.rows - 1 - (int)blockIdx.y, tid = threadIdx.x;
  const int c0 = blockIdx.x * kBlock * iters, c1 = min(a.V, c0 + kBlock * iters);
  if (c0 >= c1) return;
  const __half* x = z + (size_t)row * ldz;
  const float* tops = z_top + (size_t)row * ((a.V + 63) / 64);
  bf16* out = reinterpret_cast<bf16*>(a.dz) + (size_t)row * a.ld;
  // both pitches cover whole groups of 8 columns, so the last group of a row is read and written whole
  auto fetch = [&](uint4 (&buf)[kEach], float (&top)[kEach], int c) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int col = c + (tid + i * 256) * 8;
      if (col < c1) {
        buf[i] = __ldg(reinterpret_cast<const uint4*>(x + col));
        top[i] = __ldg(tops + col / 64);
      }
    }
  };
  uint4 cur[kEach];
  float top[kEach];
  fetch(cur, top, c0);
  float gl;
  bool live;
  const HeadCoef k = head_coef<DISTILL>(a, row, gl, live);
  if (DISTILL && blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) *a.unit = k.unit;
  const f2 cc = pack2(k.c, k.c), nl = pack2(-k.l2st, -k.l2st), A2 = pack2(k.A, k.A), B2 = pack2(k.B, k.B);
  const bool one = DISTILL && a.tau == 1.f;           // both softmaxes are the same
  const float g_kd = one ? k.g_kd + k.g_ce : k.g_kd;
  const f2 c1v = pack2(kLog2e, kLog2e), nl1 = pack2(-k.l2s1, -k.l2s1), gk = pack2(g_kd, g_kd), gc = pack2(k.g_ce, k.g_ce);
  auto value2 = [&](uint32_t h, f2 below) {           // below: the group's largest logit minus the row's
    // a distance past fp16's range counts as its end: the exponential is zero there, and 0 * l has to stay finite
    const float2 zf = __half22float2(__hmax2_nan(*reinterpret_cast<const __half2*>(&h), __floats2half2_rn(-65504.f, -65504.f)));
    const f2 d = add2(pack2(zf.x, zf.y), below), l = fma2(d, cc, nl);
    float l0, l1, r0, r1;
    unpack2(l, l0, l1);
    const f2 q = pack2(exp2_fast(l0), exp2_fast(l1));
    if (DISTILL && one) {
      unpack2(mul2(q, gk), r0, r1);
    } else if (DISTILL) {
      float e0, e1;
      unpack2(fma2(d, c1v, nl1), e0, e1);
      unpack2(fma2(gk, q, mul2(gc, pack2(exp2_fast(e0), exp2_fast(e1)))), r0, r1);
    } else {
      unpack2(mul2(q, fma2(B2, l, A2)), r0, r1);
    }
    const __nv_bfloat162 o = __floats2bfloat162_rn(r0, r1);
    return *reinterpret_cast<const uint32_t*>(&o);
  };
  for (int c = c0; c < c1; c += kBlock) {
    uint4 nxt[kEach];
    float ntop[kEach];
    if (c + kBlock < c1) fetch(nxt, ntop, c + kBlock);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int col = c + (tid + i * 256) * 8;
      if (col < c1) {
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (live) {
          const f2 below = pack2(top[i] - k.m, top[i] - k.m);
          w = make_uint4(value2(cur[i].x, below), value2(cur[i].y, below), value2(cur[i].z, below), value2(cur[i].w, below));
        }
        *reinterpret_cast<uint4*>(out + col) = w;
      }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) { cur[i] = nxt[i]; top[i] = ntop[i]; }
  }
  __syncthreads();
  if (DISTILL) distill_listed(a, k, row, c0, c1, tid, 256);
  else if (tid == 0) prob_listed(a, k, gl, row, c0, c1);
}

template <bool DISTILL>
int launch_grad_kept(const HeadFix& a, const void* z, int64_t ldz, const float* z_top, cudaStream_t st) {
  if (a.rows <= 0) return 0;
  if (a.rows > 65535 || (ldz & 7) || (a.ld & 7) || ldz < (a.V + 7) / 8 * 8 || a.ld < (a.V + 7) / 8 * 8) return 6;
  const int blocks = (a.V + 8191) / 8192;
  // as in row_grad; 16384 x 65536: 1331 us with one block per CTA, 1057 with two, 894 with four, 858 with eight
  // (811 since it computes on pairs)
  int iters = 1;
  while (iters < 8 && iters < blocks && (int64_t)a.rows * blocks >= 2ll * iters * 4 * 148) iters *= 2;
  head_grad_kept_kernel<DISTILL><<<dim3((blocks + iters - 1) / iters, a.rows), 256, 0, st>>>(a, static_cast<const __half*>(z), ldz, z_top, iters);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

}  // namespace

namespace {

// No more rows than SMs: a row is a matter of latency and takes the larger CTA (one bf16 row of 65536: 7.1 us with 512
// threads, 12.4 with 128).  Many rows: small CTAs, whose starts and ends fall apart (4096 such rows: 90 us with 128, 98 with
// 256, 117 with 512; with 20 alternatives 119, 133 and 188 us, at the same state of the kernel).
template <typename T, RowDo kDo>
int launch_row_stats(const RowStatsArgs& a, cudaStream_t st) {
  if (a.rows <= 148) row_stats_kernel<T, kDo, kFewRowsThreads><<<a.rows, kFewRowsThreads, 0, st>>>(a);
  else row_stats_kernel<T, kDo, kManyRowsThreads><<<a.rows, kManyRowsThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

}  // namespace

int row_stats(const RowStatsArgs& a, cudaStream_t st) {
  if (a.rows <= 0) return 0;
  if (a.top_k > 0) return a.is_bf16 ? launch_row_stats<bf16, kAlternatives>(a, st) : launch_row_stats<float, kAlternatives>(a, st);
  if (a.row_loss != nullptr) return a.is_bf16 ? launch_row_stats<bf16, kDistill>(a, st) : launch_row_stats<float, kDistill>(a, st);
  return a.is_bf16 ? launch_row_stats<bf16, kOnlyStats>(a, st) : launch_row_stats<float, kOnlyStats>(a, st);
}

int row_grad(const RowGradArgs& a, cudaStream_t st) {
  if (a.rows <= 0) return 0;
  const int E = a.is_bf16 ? 8 : 4;
  const int units = (a.V + 2 * E - 2) / E;            // the most a row can touch, whatever its alignment
  const int blocks = (units + kThreads * kUnroll - 1) / (kThreads * kUnroll);
  // up to four blocks per CTA while that leaves a wave of CTAs (4096 bf16 rows of 65536: 230 us with one, 180 with two, 163 with
  // four, 164 with eight; 256 rows: 12.8, 11.6, 11.6, 19.4; 16 rows: 3.7, 4.7, 6.7, 11.2)
  int iters = 1;
  while (iters < 4 && iters < blocks && (int64_t)a.rows * blocks >= 2ll * iters * 4 * 148) iters *= 2;
  const int parts = (blocks + iters - 1) / iters;
  // the grid's second axis ends at 65535 rows
  for (int r0 = (a.rows - 1) / 65535 * 65535; r0 >= 0; r0 -= 65535) {
    RowGradArgs b = a;
    b.rows = a.rows - r0 < 65535 ? a.rows - r0 : 65535;
    const size_t es = a.is_bf16 ? 2 : 4;
    b.logits = static_cast<const char*>(a.logits) + (size_t)r0 * a.ld * es;
    b.dlogits = static_cast<char*>(a.dlogits) + (size_t)r0 * a.ldd * es;
    b.stats = a.stats + r0;
    b.ids = a.ids + (size_t)r0 * a.K;
    b.w = a.w + (size_t)r0 * a.K;
    if (a.entropy != nullptr) b.entropy = a.entropy + r0;
    if (a.g_entropy != nullptr) b.g_entropy = a.g_entropy + r0;
    if (a.mask != nullptr) b.mask = a.mask + r0;
    const dim3 grid(parts, b.rows);
    if (a.g_entropy != nullptr) {
      if (a.is_bf16) row_grad_kernel<bf16, true><<<grid, kThreads, 0, st>>>(b, iters);
      else row_grad_kernel<float, true><<<grid, kThreads, 0, st>>>(b, iters);
    } else {
      if (a.is_bf16) row_grad_kernel<bf16, false><<<grid, kThreads, 0, st>>>(b, iters);
      else row_grad_kernel<float, false><<<grid, kThreads, 0, st>>>(b, iters);
    }
  }
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

int teacher_prepare(const int* ids, const void* logits, bool logits_bf16, int rows, int K, int V, float inv_tau, int* out_ids,
                    float* out_p, float2* out_row, uint16_t* first, cudaStream_t st) {
  if (rows <= 0) return 0;
  const int smem = 8 * 2 * K * (int)sizeof(int);
  if (logits_bf16)
    teacher_prepare_kernel<bf16><<<(rows + 7) / 8, 256, smem, st>>>(ids, (const bf16*)logits, rows, K, V, inv_tau, out_ids, out_p, out_row,
                                                                  first);
  else
    teacher_prepare_kernel<float><<<(rows + 7) / 8, 256, smem, st>>>(ids, (const float*)logits, rows, K, V, inv_tau, out_ids, out_p, out_row,
                                                                  first);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

int row_totals(const RowTotalsArgs& a, cudaStream_t st) {
  row_totals_kernel<<<a.count, 1024, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

int head_prob_combine(const float4* tiles, int ntiles, const int* target, const float* target_z, int rows, int V, float tau,
                      float* logprob, float* entropy, float4* stat, cudaStream_t st) {
  if (rows <= 0) return 0;
  head_prob_combine_kernel<<<(rows + 7) / 8, 256, 0, st>>>(tiles, ntiles, target, target_z, rows, V, 1.f / tau, logprob, entropy, stat);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

int head_distill_combine(const float4* tiles, int ntiles, const HeadDistillRows& a, cudaStream_t st) {
  if (a.rows <= 0) return 0;
  head_distill_combine_kernel<<<(a.rows + 7) / 8, 256, 0, st>>>(tiles, ntiles, a);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

int head_prob_fix(const HeadFix& a, cudaStream_t st) {
  if (a.rows <= 0) return 0;
  head_prob_fix_kernel<<<(a.rows + 255) / 256, 256, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

int head_distill_fix(const HeadFix& a, cudaStream_t st) {
  if (a.rows <= 0) return 0;
  head_distill_fix_kernel<<<(a.rows + 7) / 8, 256, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

int head_prob_grad_kept(const HeadFix& a, const void* z, int64_t ldz, const float* z_top, cudaStream_t st) {
  return launch_grad_kept<false>(a, z, ldz, z_top, st);
}

int head_distill_grad_kept(const HeadFix& a, const void* z, int64_t ldz, const float* z_top, cudaStream_t st) {
  return launch_grad_kept<true>(a, z, ldz, z_top, st);
}

}  // namespace rk
