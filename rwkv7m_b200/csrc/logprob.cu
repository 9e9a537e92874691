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
#include <climits>

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

// Once per row, so in 64 bits: the build's fast-math logarithm loses half the digits close to 1.
__device__ __forceinline__ float log2_row(float s) { return (float)log2((double)s); }

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
constexpr int kCandidates = 1024;

// Forward: one CTA per row.  Every thread keeps the statistics of its units and, for the alternatives, its largest logit
// and the first unit that holds it.  The k-th largest of the 256 thread maxima bounds the k-th largest column from
// below, so only the k threads above the bound are looked at again (k 256-element groups of a 65536-wide row, from L2).
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) row_stats_kernel(RowStatsArgs a) {
  constexpr int E = Row<T>::E;
  constexpr int SH = sizeof(T) == 2 ? 16 : 0;     // bf16 orders by the upper half of the key
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Row<T> r(reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld, a.V);
  const float c = kLog2e * a.inv_tau;
  if (a.mask != nullptr && a.mask[row] == 0.f) {
    // a row that does not count is not read: whatever it holds stays out of the sums
    if (tid == 0) {
      a.stats[row] = make_float2(0.f, 0.f);
      if (a.row_loss != nullptr) a.row_loss[row] = 0.f;
    }
    return;
  }

  Stat st{-INFINITY, 0.f, 0.f};
  int bu = tid;
  auto take = [&](int u, const float (&v)[E]) {
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
  };
  // first and last unit may be partly outside the row; the whole ones between them are loaded kUnroll at a time
  const int u_begin = r.whole(0) ? 0 : 1, u_end = r.whole(r.units - 1) ? r.units : r.units - 1;
  if (u_begin == 1 && tid == 0) { float v[E]; r.load(0, v); take(0, v); }
  for (int u = tid; u < u_end; u += kUnroll * kThreads) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int ui = u + i * kThreads;
      if (ui >= u_begin && ui < u_end) raw[i] = *reinterpret_cast<const uint4*>(r.x + r.first(ui));
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int ui = u + i * kThreads;
      if (ui >= u_begin && ui < u_end) { float v[E]; Row<T>::unpack(raw[i], v); take(ui, v); }
    }
  }
  if (u_end < r.units && r.units > 1 && tid == (r.units - 1) % kThreads) { float v[E]; r.load(r.units - 1, v); take(r.units - 1, v); }

  __shared__ Stat sm_stat[kThreads / 32];
  Stat tot = st;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) tot = merge(tot, shfl_xor(tot, o), c);
  if (lane == 0) sm_stat[warp] = tot;
  __syncthreads();
  tot = sm_stat[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) tot = merge(tot, sm_stat[w], c);
  const float m = tot.m;
  const float l2s = log2_row(tot.s1);                 // -inf for a row without a number, NaN for a row with one
  const float ln_s = tot.s1 > 0.f ? l2s * kLn2 : __int_as_float(0x7fffffff);
  if (tid == 0) {
    a.stats[row] = make_float2(m, l2s);
    if (a.entropy != nullptr) a.entropy[row] = tot.s1 > 0.f ? ln_s - kLn2 * (tot.s2 / tot.s1) : ln_s;
    if (a.logprob != nullptr) {
      const int id = a.ids[row];
      // an id outside the vocabulary is no token: nothing to score
      a.logprob[row] = (id >= 0 && id < a.V) ? (to_float(r.x[id]) - m) * a.inv_tau - ln_s : 0.f;
    }
  }
  if (a.row_loss != nullptr) {
    // distillation: mask tau^2 (sum p ln p - sum p ln q) over the teacher's alternatives
    float acc = 0.f;
    for (int j = tid; j < a.K; j += kThreads) {
      const float p = a.t_prob[(size_t)row * a.K + j];
      const int id = a.t_ids[(size_t)row * a.K + j];
      if (p > 0.f) acc += p * ((to_float(r.x[id]) - m) * a.inv_tau - ln_s);
    }
    acc = warp_sum(acc);
    __shared__ float sm_acc[kThreads / 32];
    if (lane == 0) sm_acc[warp] = acc;
    __syncthreads();
    if (tid == 0) {
      float s = 0.f;
      for (int w = 0; w < kThreads / 32; ++w) s += sm_acc[w];
      const float2 t = a.t_row[row];                  // sum p ln p, and 1 or 0 for a row without alternatives
      a.row_loss[row] = t.y > 0.f ? (a.mask != nullptr ? a.mask[row] : 1.f) * a.tau * a.tau * (t.x - s) : 0.f;
    }
  }
  if constexpr (TOP) {
    __shared__ int sm_sel[kThreads], sm_nsel, sm_n;
    __shared__ uint2 sm_cand[kCandidates];
    const int k = a.top_k;
    const uint32_t key = tid < r.units ? order_key(st.m) >> SH : 0u;     // a thread without units has none
    // largest bound that at least k thread maxima reach; among equal ones the lowest units
    uint32_t bound = 0u;
    for (int b = 31 - SH; b >= 0; --b) {
      const uint32_t t = bound | (1u << b);
      if (__syncthreads_count(key >= t) >= k) bound = t;
    }
    const int above = __syncthreads_count(key > bound), equal = __syncthreads_count(key == bound && tid < r.units);
    int last = INT_MAX;                               // equal maxima count up to this unit
    if (bound > 0u && above + equal > k) {
      last = 0;
      for (int b = 30; b >= 0; --b)                   // smallest unit with enough equal maxima at or below it, minus one
        if (__syncthreads_count(key == bound && bu < (last | (1 << b))) < k - above) last |= 1 << b;
    }
    if (tid == 0) { sm_nsel = 0; sm_n = 0; }
    for (int i = tid; i < k; i += kThreads) {
      a.top_ids[(size_t)row * k + i] = -1;            // stays where the row has fewer than k numbers
      a.top_logprobs[(size_t)row * k + i] = __int_as_float(0x7fffffff);
    }
    __syncthreads();
    if (tid < r.units && (key > bound || (key == bound && bu <= last))) sm_sel[atomicAdd(&sm_nsel, 1)] = tid;
    __syncthreads();
    const int nsel = sm_nsel, per = (r.units + kThreads - 1) / kThreads;
    // every element of the chosen threads' units, in any order
    auto each = [&](auto&& f) {
      for (int i = tid; i < nsel * per; i += kThreads) {
        const int uu = sm_sel[i % nsel] + (i / nsel) * kThreads;
        if (uu >= r.units) continue;
        float v[E];
        r.load(uu, v);
        const int i0 = r.first(uu);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int idx = i0 + e;
          if (idx >= 0 && idx < a.V && v[e] == v[e]) f(order_key(v[e]) >> SH, idx, uu, v[e]);
        }
      }
    };
    each([&](uint32_t kk, int idx, int uu, float v) {
      if (kk > bound || (kk == bound && uu <= last)) {
        const int at = atomicAdd(&sm_n, 1);
        if (at < kCandidates) sm_cand[at] = make_uint2(__float_as_uint(v), (uint32_t)idx);
      }
    });
    __syncthreads();
    int n = sm_n;
    __syncthreads();
    if (n > kCandidates) {
      // a row whose chosen threads hold long runs above the bound (sorted or blockwise data): the exact k-th element of
      // them, by bisection over the value and then over the index
      uint32_t kth = 0u;
      for (int b = 31 - SH; b >= 0; --b) {
        const uint32_t t = kth | (1u << b);
        int cnt = 0;
        each([&](uint32_t kk, int, int, float) { cnt += kk >= t; });
        if (tid == 0) sm_n = 0;
        __syncthreads();
        atomicAdd(&sm_n, cnt);
        __syncthreads();
        if (sm_n >= k) kth = t;
        __syncthreads();
      }
      int gt = 0;
      each([&](uint32_t kk, int, int, float) { gt += kk > kth; });
      if (tid == 0) sm_n = 0;
      __syncthreads();
      atomicAdd(&sm_n, gt);
      __syncthreads();
      const int need = k - sm_n;
      __syncthreads();
      int lim = 0;                                    // elements equal to the k-th count below this index, inclusive
      for (int b = 30; b >= 0; --b) {
        int cnt = 0;
        each([&](uint32_t kk, int idx, int, float) { cnt += kk == kth && idx < (lim | (1 << b)); });
        if (tid == 0) sm_n = 0;
        __syncthreads();
        atomicAdd(&sm_n, cnt);
        __syncthreads();
        if (sm_n < need) lim |= 1 << b;
        __syncthreads();
      }
      if (tid == 0) sm_n = 0;
      __syncthreads();
      each([&](uint32_t kk, int idx, int, float v) {
        if (kk > kth || (kk == kth && idx <= lim)) {
          const int at = atomicAdd(&sm_n, 1);
          if (at < kCandidates) sm_cand[at] = make_uint2(__float_as_uint(v), (uint32_t)idx);
        }
      });
      __syncthreads();
      n = min(sm_n, kCandidates);
    }
    for (int i = tid; i < n; i += kThreads) {
      const float v = __uint_as_float(sm_cand[i].x);
      const uint32_t idx = sm_cand[i].y;
      int rank = 0;
      for (int j = 0; j < n; ++j) {
        const float w = __uint_as_float(sm_cand[j].x);
        rank += w > v || (w == v && sm_cand[j].y < idx);
      }
      if (rank < k) {
        a.top_ids[(size_t)row * k + rank] = (int)idx;
        a.top_logprobs[(size_t)row * k + rank] = (v - m) * a.inv_tau - ln_s;
      }
    }
  }
}

// Backward: one CTA per kThreads * kUnroll units of a row.  Dense part first, then the columns of the sparse list that lie
// in this CTA's part are written again with their whole value (the list may name a column more than once).
template <typename T>
__global__ void __launch_bounds__(kThreads) row_grad_kernel(RowGradArgs a) {
  constexpr int E = Row<T>::E;
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld;
  T* out = reinterpret_cast<T*>(a.dlogits) + (size_t)row * a.ldd;
  const Row<T> o(out, a.V);                           // units by the output's alignment
  const int u0 = blockIdx.x * kThreads * kUnroll;
  if (u0 >= o.units) return;
  float scale = a.weight_mul;
  if (a.g_scale != nullptr) scale *= a.g_scale[0];
  if (a.mask != nullptr) scale = a.mask[row] == 0.f ? 0.f : scale * a.mask[row];
  const float g_h = a.g_entropy != nullptr ? a.g_entropy[row] : 0.f;
  __shared__ float sm_w[kThreads / 32];
  __shared__ int sm_any;
  float wsum = 0.f;
  int any = g_h != 0.f;
  if (scale != 0.f)
    for (int j = tid; j < a.K; j += kThreads) {
      const int id = a.ids[(size_t)row * a.K + j];
      const float w = a.w[(size_t)row * a.K + j];
      if (id >= 0 && id < a.V && w != 0.f) { wsum += w; any = 1; }
    }
  any = __syncthreads_or(any);
  wsum = warp_sum(wsum);
  if (lane == 0) sm_w[warp] = wsum;
  __syncthreads();
  wsum = 0.f;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) wsum += sm_w[w];
  const float2 st = a.stats[row];
  const float c = kLog2e * a.inv_tau;
  const float m = st.x, l2s = st.y;
  const float A = any ? a.inv_tau * (-scale * wsum - (g_h != 0.f ? g_h * a.entropy[row] : 0.f)) : 0.f;
  const float B = -g_h * a.inv_tau * kLn2;            // times log2 q
  auto value = [&](float z) {
    float t = (z - m) * c - l2s;
    t = t < kMinExponent ? kMinExponent : t;
    return exp2_fast(t) * fmaf(B, t, A);
  };
  const bool congruent = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const Row<T> r(x, a.V);
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int u = u0 + tid + i * kThreads;
    if (u >= o.units) break;
    const int i0 = o.first(u);
    float v[E];
    if (!any) {
      // nothing flows into this row (padding, a masked row): its logits are not read, so they may hold anything
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = 0.f;
    } else {
      if (congruent) r.load(u, v);
      else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = (i0 + e >= 0 && i0 + e < a.V) ? to_float(x[i0 + e]) : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = value(v[e]);
    }
    if (o.whole(u)) {
      uint4 raw;
      if constexpr (sizeof(T) == 2) {
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      } else {
        raw = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      }
      *reinterpret_cast<uint4*>(out + i0) = raw;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) if (i0 + e >= 0 && i0 + e < a.V) out[i0 + e] = from_float<T>(v[e]);
    }
  }
  if (!any) return;
  __syncthreads();
  const int lo = o.first(u0), hi = o.first(u0 + kThreads * kUnroll);
  for (int j = tid; j < a.K; j += kThreads) {
    const int id = a.ids[(size_t)row * a.K + j];
    if (id < 0 || id >= a.V || id < lo || id >= hi) continue;
    float w = 0.f;
    for (int i = 0; i < a.K; ++i) if (a.ids[(size_t)row * a.K + i] == id) w += a.w[(size_t)row * a.K + i];
    out[id] = from_float<T>(value(to_float(x[id])) + scale * w * a.inv_tau);
  }
}

// A teacher's alternatives, one warp per row: p = softmax of their logits / tau over those that are there (id inside the
// vocabulary, logit above -inf), sorted by id so that a pass over the columns in order meets them in order; absent ones
// go last with the id INT_MAX and p = 0.  Also sum p ln p and whether the row has any.
template <typename T>
__global__ void __launch_bounds__(256) teacher_prepare_kernel(const int* __restrict__ ids, const T* __restrict__ logits,
                                                              int rows, int K, int V, float inv_tau, int* __restrict__ out_ids,
                                                              float* __restrict__ out_p, float2* __restrict__ out_row) {
  extern __shared__ int sm_ids[];                     // [8][K]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x * 8 + warp;
  if (row >= rows) return;
  int* my = sm_ids + warp * K;
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
    out_ids[(size_t)row * K + rank] = id;
    out_p[(size_t)row * K + rank] = id != INT_MAX ? exp2_fast(fmaxf((to_float(rl[j]) - m) * c, kMinExponent)) * inv : 0.f;
  }
  if (lane == 0) out_row[row] = s > 0.f ? make_float2(kLn2 * (s2 * inv - log2_row(s)), 1.f) : make_float2(0.f, 0.f);
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

__global__ void __launch_bounds__(256) head_prob_fix_kernel(HeadFix a) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= a.rows || a.g0 == nullptr) return;
  const int id = a.target[row];
  const float gl = a.g0[row], gh = a.g1 != nullptr ? a.g1[row] : 0.f;
  if (id < 0 || id >= a.V || gl == 0.f) return;
  const float inv_tau = 1.f / a.tau;
  const float4 s = a.stat[row];
  const float l = (a.target_z[row] - s.x) * (kLog2e * inv_tau) - s.z;
  const float A = inv_tau * (-gl - (gh != 0.f ? gh * s.w : 0.f)), B = -gh * inv_tau * kLn2;
  reinterpret_cast<bf16*>(a.dz)[(size_t)row * a.ld + id] = f2bf(fmaf(exp2_fast(l), fmaf(B, l, A), gl * inv_tau));
}

// One warp per row.  The teacher's ids are sorted, so equal ones are neighbours and the first of a run writes for all.
__global__ void __launch_bounds__(256) head_distill_fix_kernel(HeadFix a) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= a.rows) return;
  const float inv_tau = 1.f / a.tau, c = kLog2e * inv_tau;
  const float4 s = a.stat[row];
  const float2 w = a.weight[row];
  const float g_ce = a.g0 != nullptr ? a.g0[0] * w.x : 0.f, g_kd = a.g1 != nullptr ? a.g1[0] * w.y * a.tau : 0.f;
  const float g_l2 = a.g_l2 != nullptr ? a.g_l2[0] * 1e-4f * s.x : 0.f;
  const int tgt = w.x != 0.f ? a.target[row] : -1, am = a.argmax[row];
  bf16* dz = reinterpret_cast<bf16*>(a.dz) + (size_t)row * a.ld;
  auto value = [&](int col, float z, float p) {
    float d = 0.f;
    if (g_kd != 0.f) d = g_kd * (exp2_fast((z - s.x) * c - s.z) - p);
    if (g_ce != 0.f) d += g_ce * (exp2_fast((z - s.x) * kLog2e - s.y) - (col == tgt ? 1.f : 0.f));
    if (col == am) d += g_l2;
    return f2bf(d);
  };
  bool tgt_done = tgt < 0, am_done = false;
  for (int j0 = 0; j0 < a.K; j0 += 32) {
    const int j = j0 + lane;
    const size_t at = (size_t)row * a.K + j;
    const int id = j < a.K ? a.t_ids[at] : INT_MAX;
    if (id != INT_MAX && (j == 0 || a.t_ids[at - 1] != id)) {
      float p = a.t_prob[at];
      for (int i = 1; j + i < a.K && a.t_ids[at + i] == id; ++i) p += a.t_prob[at + i];
      dz[id] = value(id, a.cols_z[at], p);
    }
    tgt_done = tgt_done || __any_sync(0xffffffffu, id == tgt);
    am_done = am_done || __any_sync(0xffffffffu, id == am);
  }
  if (lane == 0 && !tgt_done) dz[tgt] = value(tgt, a.target_z[row], 0.f);
  if (lane == 0 && !am_done && am != tgt && am >= 0 && am < a.V) dz[am] = value(am, s.x, 0.f);
}

}  // namespace

int row_stats(const RowStatsArgs& a, cudaStream_t st) {
  if (a.rows <= 0) return 0;
  if (a.top_k > 0) {
    if (a.is_bf16) row_stats_kernel<bf16, true><<<a.rows, kThreads, 0, st>>>(a);
    else row_stats_kernel<float, true><<<a.rows, kThreads, 0, st>>>(a);
  } else {
    if (a.is_bf16) row_stats_kernel<bf16, false><<<a.rows, kThreads, 0, st>>>(a);
    else row_stats_kernel<float, false><<<a.rows, kThreads, 0, st>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

int row_grad(const RowGradArgs& a, cudaStream_t st) {
  if (a.rows <= 0) return 0;
  const int E = a.is_bf16 ? 8 : 4;
  const int units = (a.V + 2 * E - 2) / E;            // the most a row can touch, whatever its alignment
  const int parts = (units + kThreads * kUnroll - 1) / (kThreads * kUnroll);
  // the grid's second axis ends at 65535 rows
  for (int r0 = 0; r0 < a.rows; r0 += 65535) {
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
    if (a.is_bf16) row_grad_kernel<bf16><<<dim3(parts, b.rows), kThreads, 0, st>>>(b);
    else row_grad_kernel<float><<<dim3(parts, b.rows), kThreads, 0, st>>>(b);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

int teacher_prepare(const int* ids, const void* logits, bool logits_bf16, int rows, int K, int V, float inv_tau, int* out_ids,
                    float* out_p, float2* out_row, cudaStream_t st) {
  if (rows <= 0) return 0;
  const int smem = 8 * K * (int)sizeof(int);
  if (logits_bf16)
    teacher_prepare_kernel<bf16><<<(rows + 7) / 8, 256, smem, st>>>(ids, (const bf16*)logits, rows, K, V, inv_tau, out_ids, out_p, out_row);
  else
    teacher_prepare_kernel<float><<<(rows + 7) / 8, 256, smem, st>>>(ids, (const float*)logits, rows, K, V, inv_tau, out_ids, out_p, out_row);
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

}  // namespace rk
