// Router with the quantities that training and load monitoring need, in one pass over the logits:
//   a = l (softmax) or log sigmoid(l);  p = softmax(a)   -- for sigmoid scores that is sigmoid(l) / sum sigmoid(l), free of
//                                                           0/0 where every score underflows
//   ids: the K largest logits, equal ones in ascending expert order;  weights: p (or sigmoid) of them, or the softmax of
//   a over the chosen experts (renormalised)
//   counts[s,e] = how often expert e was chosen by the live tokens of sequence s
//   balance = mean over the sequences with n_s > 0 live tokens of  E / (K n_s^2) sum_e counts[s,e] sum_t p[t,e]
//   z = mean over the live tokens of logsumexp(l)^2
// A token is live if its mask entry is set, it lies inside a sequence, and not all of its logits are -inf.  Others get
// ids 0..K-1, weights 0 and gradient 0, whatever their logits hold.
//
// The logits are a few MB at most, so latency bounds it: a row is held by 8, 16 or 32 lanes, and a CTA takes a chunk of
// consecutive rows.  Sums over tokens: a chunk and a sequence that overlap write one row of partial sums at slot
// chunk + sequence -- the overlapping pairs form a staircase, so no two share a slot -- and a second launch adds the
// slots of a sequence in order.  No atomics on floats: the same bits on every run.
// On a B200: 64 x 128 experts, top 4: 3.7 + 4.1 us; 16384 x 8, top 2: 4.7 + 6.9, backward 3.4 us; 4096 x 256, top 8: 10.1 + 7.3,
// backward 8.4 us, with sigmoid scores, a mask and 13 sequences 16.0 + 6.1 and 10.4 us; 16384 x 256: 29 + 8.6, 17.7 us (the
// selection's instructions).  A launch with a single row takes 5 us.
#include <algorithm>

#include "rowwise.cuh"

namespace b200moe {

namespace {

constexpr int kRouterThreads = 256;
constexpr int kRouterWarps = kRouterThreads / 32;
constexpr int kMaxExperts = 1024, kMaxRouterTopk = 32;

struct RouterParams {
  const void* logits;
  int64_t stride;
  const uint8_t* mask;
  const int32_t* cu;          // [S + 1] or null (one sequence of all tokens)
  float* weights;
  int32_t* ids;
  float* lse;                 // [2, T]: logsumexp of a and of l (backward), or null
  int32_t* seg;               // [T]: sequence of a live token, -1 otherwise (backward), or null
  float* part_p;              // [slots, E]
  int32_t* part_c;            // [slots, E]
  float* part_z;              // [slots]: sum of logsumexp^2
  int32_t* part_n;            // [slots]: live tokens
  int32_t* ticket;
  int T, E, K, S, rows, scoring, renorm;
};

// Order keys of the logits: ascending unsigned order = ascending float order, NaN above everything, the two zeros alike, and
// 0 = taken (no value has it).  A 16-bit logit leaves room for its expert: one maximum then finds both, the lowest expert
// first among equal logits; a 32-bit one needs a second reduction over the experts that hold the maximum.
template <typename T> constexpr bool kKeyHoldsExpert = sizeof(T) == 2;
__device__ __forceinline__ uint32_t order32(uint32_t u) {
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (u == 0x80000000u) u = 0u;
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint32_t order_key(float v, int) { return order32(__float_as_uint(v)); }
__device__ __forceinline__ uint32_t order16(uint32_t u, uint32_t inf) {
  if ((u & 0x7fffu) > inf) return 0xffffu;
  if (u == 0x8000u) u = 0u;
  return u ^ ((u >> 15) ? 0xffffu : 0x8000u);
}
__device__ __forceinline__ uint32_t order_key(__nv_bfloat16 v, int e) {
  return (order16(__bfloat16_as_ushort(v), 0x7f80u) << 16) | (0xffffu - (uint32_t)e);
}
__device__ __forceinline__ uint32_t order_key(__half v, int e) {
  return (order16(__half_as_ushort(v), 0x7c00u) << 16) | (0xffffu - (uint32_t)e);
}
// the logit of a key
template <typename T> __device__ __forceinline__ float key_value(uint32_t k);
template <> __device__ __forceinline__ float key_value<float>(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
template <> __device__ __forceinline__ float key_value<__nv_bfloat16>(uint32_t k) {
  k >>= 16;
  return __uint_as_float((k ^ ((k >> 15) ? 0x8000u : 0xffffu)) << 16);
}
template <> __device__ __forceinline__ float key_value<__half>(uint32_t k) {
  k >>= 16;
  return __half2float(__ushort_as_half((unsigned short)(k ^ ((k >> 15) ? 0x8000u : 0xffffu))));
}
template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int d = LPR / 2; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
template <int LPR>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  if constexpr (LPR == 32) return __reduce_max_sync(0xffffffffu, v);
#pragma unroll
  for (int d = LPR / 2; d > 0; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
template <int LPR>
__device__ __forceinline__ uint32_t group_min(uint32_t v) {
  if constexpr (LPR == 32) return __reduce_min_sync(0xffffffffu, v);
#pragma unroll
  for (int d = LPR / 2; d > 0; d >>= 1) v = min(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
// a maximum that NaN survives
__device__ __forceinline__ float max_nan(float a, float b) { return (a != a || b != b) ? __uint_as_float(0x7fc00000u) : fmaxf(a, b); }
template <int LPR>
__device__ __forceinline__ float group_max_nan(float v) {
#pragma unroll
  for (int d = LPR / 2; d > 0; d >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

// A row's scores up to the factor exp(shift): softmax exp(l - max) with shift = max; sigmoid 1 / (1 + exp(-l)) with shift = 0,
// or, where every logit is negative, exp(l - max) / (1 + exp(l)) with shift = max, which cannot underflow for all of them.
struct RowScore {
  float lmax;
  bool sigmoid, shifted;
  __device__ RowScore(float lmax_, bool sigmoid_) : lmax(lmax_), sigmoid(sigmoid_), shifted(!sigmoid_ || lmax_ < 0.f) {}
  __device__ __forceinline__ float shift() const { return shifted ? lmax : 0.f; }
  // score of l, and exp(l - max) in `el`
  __device__ __forceinline__ float operator()(float l, float& el) const {
    el = expf(l - lmax);
    if (!sigmoid) return el;
    if (shifted) return __fdividef(el, 1.f + expf(l));
    const float t = expf(-fabsf(l));
    return __fdividef(l >= 0.f ? 1.f : t, 1.f + t);
  }
};

__device__ __forceinline__ int clamp_row(int v, int T) { return min(max(v, 0), T); }

template <typename T, int LPR, int VPL>
__global__ void __launch_bounds__(kRouterThreads)
router_forward_kernel(const __grid_constant__ RouterParams p) {
  extern __shared__ float smem[];                       // [warps][E] sums of p, [E] counts
  __shared__ float warp_z[kRouterWarps];
  __shared__ int32_t warp_n[kRouterWarps];
  grid_dep_wait();
  grid_dep_launch();
  const int E = p.E, K = p.K;
  float* sum_p = smem;
  int32_t* cnt = reinterpret_cast<int32_t*>(smem + kRouterWarps * E);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / LPR, l0 = lane % LPR;
  constexpr int RPW = 32 / LPR;                         // rows of a warp at a time
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0;
  const int row0 = blockIdx.x * p.rows, row1 = min(row0 + p.rows, p.T);

  auto dead = [&](int64_t t) {                           // called by the LPR lanes of a row
    for (int k = l0; k < K; k += LPR) { p.ids[t * K + k] = k; p.weights[t * K + k] = 0.f; }
    if (l0 == 0 && p.seg != nullptr) p.seg[t] = -1;
  };

  // the first sequence that ends behind this chunk's first row
  int s = 0, at = row0;
  if (p.cu != nullptr) {
    int hi = p.S;
    while (s < hi) {
      const int mid = (s + hi) >> 1;
      if (clamp_row(p.cu[mid + 1], p.T) > row0) hi = mid; else s = mid + 1;
    }
    const int first = max(row0, min(clamp_row(p.cu[0], p.T), row1));
    for (int t = row0 + warp * RPW + sub; t < first; t += kRouterWarps * RPW) dead(t);
    at = first;
  }
  for (; s < p.S && at < row1; ++s) {
    const int end = p.cu != nullptr ? min(row1, max(at, clamp_row(p.cu[s + 1], p.T))) : row1;
    if (end == at) continue;                             // an empty sequence
    for (int e = threadIdx.x; e < E; e += kRouterThreads) cnt[e] = 0;
    __syncthreads();
    float acc[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc[i] = 0.f;
    float zsum = 0.f;
    int n = 0;
    for (int tb = at + warp * RPW; tb < end; tb += kRouterWarps * RPW) {     // uniform in the warp
      const int t = tb + sub;
      const bool row = t < end;
      const T* src = static_cast<const T*>(p.logits) + (int64_t)t * p.stride;
      float l[VPL], ex[VPL];
      uint32_t key[VPL];
      float lmax = -INFINITY;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int e = l0 + i * LPR;
        const bool in = row && e < E;
        const T v = in ? src[e] : from_f<T>(-INFINITY);
        l[i] = to_f(v);
        key[i] = in ? order_key(v, e) : 0u;
        lmax = max_nan(lmax, l[i]);
      }
      bool live = row && (p.mask == nullptr || p.mask[t] != 0);
      lmax = group_max_nan<LPR>(lmax);
      live = live && lmax != -INFINITY;
      const RowScore score(lmax, p.scoring != 0);
      float sum = 0.f, sum_l = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        float el;
        ex[i] = score(l[i], el);
        sum += ex[i];
        sum_l += el;
      }
      sum = group_sum<LPR>(sum);
      sum_l = p.scoring == 0 ? sum : group_sum<LPR>(sum_l);
      const float inv = 1.f / sum;
      const float lse_a = score.shift() + logf(sum), lse_l = lmax + logf(sum_l);
      // lane k of the row keeps the k-th choice
      uint32_t my_key = 0u;
      int id = 0;
      for (int k = 0; k < K; ++k) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < VPL; ++i) best = max(best, key[i]);
        best = group_max<LPR>(best);
        int e;
        if constexpr (kKeyHoldsExpert<T>) {
          e = (int)(0xffffu - (best & 0xffffu));
#pragma unroll
          for (int i = 0; i < VPL; ++i) key[i] = key[i] == best ? 0u : key[i];
        } else {
          uint32_t mine = 0x7fffffffu;                   // lowest expert of this lane that holds the best key
#pragma unroll
          for (int i = VPL - 1; i >= 0; --i)
            if (key[i] == best) mine = (uint32_t)(l0 + i * LPR);
          const uint32_t first = group_min<LPR>(mine);
          e = (int)first;
#pragma unroll
          for (int i = 0; i < VPL; ++i)
            if (first == (uint32_t)(l0 + i * LPR)) key[i] = 0u;
        }
        if (l0 == k) { my_key = best; id = e; }
      }
      float chosen = 0.f, unused;
      if (l0 < K) chosen = score(key_value<T>(my_key), unused);
      const float total = group_sum<LPR>(chosen);
      if (live) {
        if (l0 < K) {
          const float w = p.renorm ? chosen / total : (p.scoring == 0 ? chosen * inv : chosen * expf(score.shift()));
          p.ids[(int64_t)t * K + l0] = id;
          p.weights[(int64_t)t * K + l0] = w;
          atomicAdd(&cnt[id], 1);
        }
        if (l0 == 0) {
          if (p.lse != nullptr) { p.lse[t] = lse_a; p.lse[p.T + t] = lse_l; p.seg[t] = s; }
          zsum = fmaf(lse_l, lse_l, zsum);
          ++n;
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) acc[i] = fmaf(ex[i], inv, acc[i]);
      } else if (row) {
        dead(t);
      }
    }
    // join the rows of a warp, then the warps
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
#pragma unroll
      for (int d = LPR; d < 32; d <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], d);
      const int e = l0 + i * LPR;
      if (sub == 0 && e < E) sum_p[warp * E + e] = acc[i];
    }
    zsum = warp_sum(zsum);
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) { warp_z[warp] = zsum; warp_n[warp] = n; }
    __syncthreads();
    const int64_t slot = (int64_t)blockIdx.x + s;
    for (int e = threadIdx.x; e < E; e += kRouterThreads) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kRouterWarps; ++w) v += sum_p[w * E + e];
      p.part_p[slot * E + e] = v;
      p.part_c[slot * E + e] = cnt[e];
    }
    if (threadIdx.x == 0) {
      float z = 0.f;
      int m = 0;
      for (int w = 0; w < kRouterWarps; ++w) { z += warp_z[w]; m += warp_n[w]; }
      p.part_z[slot] = z;
      p.part_n[slot] = m;
    }
    __syncthreads();                                     // the shared sums are reused by the next sequence
    at = end;
  }
  for (int t = at + warp * RPW + sub; t < row1; t += kRouterWarps * RPW) dead(t);   // behind the last sequence
}

struct RouterJoinParams {
  const int32_t* cu;
  const float* part_p; const int32_t* part_c; const float* part_z; const int32_t* part_n;
  int32_t* ticket;
  int32_t* counts;            // [S, E]
  float* coef;                // [S, E]: E counts / (K n_s^2), the loss of the sequence = sum(coef * sum of p)
  float* seq;                 // [S, blocks, 3]: loss of the block's experts, live tokens, sum of logsumexp^2
  float* stats;               // {1 / sequences with live tokens, 1 / live tokens}
  float* balance; float* z;
  int T, E, K, S, rows, chunks;
};

// One CTA per sequence and 64 experts; the last one to finish joins the sequences in order.
constexpr int kJoinThreads = 1024, kJoinCols = 64;
__global__ void __launch_bounds__(kJoinThreads)
router_join_kernel(const __grid_constant__ RouterJoinParams p) {
  __shared__ float gp[kJoinThreads];                    // [groups][columns] sums of p, and of counts
  __shared__ int32_t gc[kJoinThreads];
  __shared__ float zs, half;
  __shared__ int ns, last;
  grid_dep_wait();
  grid_dep_launch();
  const int s = blockIdx.x, E = p.E, e0 = blockIdx.y * kJoinCols, nb = gridDim.y;
  int lo = 0, hi = p.T;
  if (p.cu != nullptr) {
    lo = clamp_row(p.cu[s], p.T);
    hi = max(lo, clamp_row(p.cu[s + 1], p.T));
  }
  const int c0 = hi > lo ? lo / p.rows : 0, c1 = hi > lo ? (hi - 1) / p.rows + 1 : 0;
  // groups of threads take interleaved slots of a column; their sums are added in order
  const int cols = min(E - e0, kJoinCols), groups = kJoinThreads / cols;
  const int g = threadIdx.x / cols, e = e0 + threadIdx.x % cols;
  if (g < groups) {
    float v = 0.f;
    int c = 0;
#pragma unroll 4
    for (int i = c0 + g; i < c1; i += groups) {
      v += p.part_p[(int64_t)(i + s) * E + e];
      c += p.part_c[(int64_t)(i + s) * E + e];
    }
    gp[threadIdx.x] = v;
    gc[threadIdx.x] = c;
  }
  if (threadIdx.x >= kJoinThreads - 32) {
    const int lane = threadIdx.x & 31;
    float z = 0.f;
    int n = 0;
#pragma unroll 4
    for (int i = c0 + lane; i < c1; i += 32) { z += p.part_z[i + s]; n += p.part_n[i + s]; }
    z = warp_sum(z);
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) { zs = z; ns = n; }
  }
  __syncthreads();
  if (threadIdx.x >= kJoinCols) return;
  const float n = (float)ns;
  const float f = ns > 0 ? (float)E / ((float)p.K * n * n) : 0.f;
  float loss = 0.f;
  if ((int)threadIdx.x < cols) {
    float v = 0.f;
    int c = 0;
    for (int i = 0; i < groups; ++i) { v += gp[i * cols + threadIdx.x]; c += gc[i * cols + threadIdx.x]; }
    const float cf = f * (float)c;
    p.counts[(int64_t)s * E + e] = c;
    if (p.coef != nullptr) p.coef[(int64_t)s * E + e] = cf;
    if (ns > 0) loss = cf * v;
  }
  loss = warp_sum(loss);
  if (threadIdx.x == 32) half = loss;
  asm volatile("bar.sync 1, 64;" ::: "memory");
  if (threadIdx.x >= 32) return;
  if (threadIdx.x == 0) {
    float* o = p.seq + ((int64_t)s * nb + blockIdx.y) * 3;
    o[0] = loss + half; o[1] = n; o[2] = zs;
    __threadfence();
    last = atomicAdd(p.ticket, 1) == (int)(gridDim.x * gridDim.y) - 1;
  }
  __syncwarp();
  if (last) {
    __threadfence();
    float tot = 0.f, tok = 0.f, z = 0.f, used = 0.f;
    for (int i = threadIdx.x; i < p.S * nb; i += 32) {
      const volatile float* o = p.seq + (int64_t)i * 3;
      tot += o[0];
      if (i % nb == 0) {
        tok += o[1]; z += o[2];
        used += o[1] > 0.f ? 1.f : 0.f;
      }
    }
    tot = warp_sum(tot); tok = warp_sum(tok); z = warp_sum(z); used = warp_sum(used);
    if (threadIdx.x == 0) {
      const float iu = 1.f / fmaxf(used, 1.f), it = 1.f / fmaxf(tok, 1.f);
      *p.balance = tot * iu;
      *p.z = z * it;
      if (p.stats != nullptr) { p.stats[0] = iu; p.stats[1] = it; }
    }
  }
}

struct RouterBwdParams {
  const void* logits;
  int64_t stride;
  const float* lse; const int32_t* seg; const int32_t* ids; const float* weights;
  const float* coef; const float* stats;
  const float* dweights; const float* dbalance; const float* dz;    // each may be null
  void* dlogits;
  int T, E, K, scoring, renorm;
};

// Per row, from the saved logsumexps, with q = dbalance coef[s] / sequences:
//   da = p (q - sum p q)  +  the weights' part, on the chosen experts: w (dw - sum w dw) renormalised, else w dw (softmax:
//   less p sum w dw everywhere);  dl = da (softmax) or da sigmoid(-l);  + 2 dz lse / tokens softmax(l)
template <typename T, int LPR, int VPL>
__global__ void __launch_bounds__(kRouterThreads)
router_backward_kernel(const __grid_constant__ RouterBwdParams p) {
  __shared__ float rows[kRouterWarps * (32 / LPR) * LPR * VPL];
  grid_dep_wait();
  grid_dep_launch();
  const int E = p.E, K = p.K;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / LPR, l0 = lane % LPR;
  constexpr int RPW = 32 / LPR;
  const bool sigmoid = p.scoring != 0;
  const float gb = p.dbalance != nullptr ? *p.dbalance * p.stats[0] : 0.f;
  const float gz = p.dz != nullptr ? 2.f * *p.dz * p.stats[1] : 0.f;
  for (int64_t tb = ((int64_t)blockIdx.x * kRouterWarps + warp) * RPW; tb < p.T; tb += (int64_t)gridDim.x * kRouterWarps * RPW) {
    const int64_t t = tb + sub;
    const bool row = t < p.T;
    const int s = row ? p.seg[t] : -1;
    const bool live = s >= 0;
    const T* src = static_cast<const T*>(p.logits) + t * p.stride;
    float l[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = l0 + i * LPR;
      l[i] = row && e < E ? to_f(src[e]) : -INFINITY;
    }
    // p = score / exp(lse - shift) as in the forward pass; m = d(a) / dl; pl = softmax(l)
    const float lse_a = live ? p.lse[t] : 0.f, lse_l = live ? p.lse[p.T + t] : 0.f;
    float w = 0.f, dw = 0.f, wdw = 0.f;                // lane k of the row holds its k-th choice
    int id = -1;
    if (live && l0 < K && p.dweights != nullptr) {
      w = p.weights[t * K + l0];
      dw = p.dweights[t * K + l0];
      id = p.ids[t * K + l0];
      wdw = w * dw;
    }
    float pr[VPL], m[VPL], q[VPL], dot = 0.f;
    const bool low = lse_a < -40.f;                    // sigmoid scores that may all underflow: in logarithms
    const float scale = expf(-lse_a);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = l0 + i * LPR;
      if (!sigmoid) {
        pr[i] = expf(l[i] - lse_a);
        m[i] = 1.f;
      } else {
        const float t1 = expf(-fabsf(l[i])), r = __fdividef(1.f, 1.f + t1);
        pr[i] = low ? expf(l[i] - lse_a) * r : (l[i] >= 0.f ? r : t1 * r) * scale;
        m[i] = l[i] >= 0.f ? t1 * r : r;
      }
      if (!live || e >= E) pr[i] = 0.f;
      q[i] = (gb != 0.f && live && e < E) ? gb * p.coef[(int64_t)s * E + e] : 0.f;
      dot = fmaf(pr[i], q[i], dot);
    }
    dot = group_sum<LPR>(dot);
    const float sum_w = group_sum<LPR>(wdw);
    const float part = p.renorm ? w * (dw - sum_w) : wdw;
    const float all = (!p.renorm && !sigmoid) ? dot + sum_w : dot;
    float da[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) da[i] = pr[i] * (q[i] - all);
    if (p.dweights != nullptr) {
      // the choices' parts, by way of a row of zeros in shared memory
      float* mine = rows + (warp * RPW + sub) * (LPR * VPL);
#pragma unroll
      for (int i = 0; i < VPL; ++i) mine[l0 + i * LPR] = 0.f;
      __syncwarp();
      if (id >= 0 && id < E) mine[id] = part;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < VPL; ++i) da[i] += mine[l0 + i * LPR];
      __syncwarp();
    }
    if (row) {
      T* dst = static_cast<T*>(p.dlogits) + t * E;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int e = l0 + i * LPR;
        if (e < E) {
          float d = da[i] * m[i];
          if (gz != 0.f) d = fmaf(gz * lse_l, sigmoid ? expf(l[i] - lse_l) : pr[i], d);
          dst[e] = from_f<T>(live ? d : 0.f);
        }
      }
    }
  }
}

// layout of the forward's workspace: partial sums by slot, the sequences' sums, the ticket
struct RouterLayout {
  int rows, chunks;
  int64_t slots, off_c, off_z, off_n, off_seq, off_ticket, bytes;
};
RouterLayout router_layout(int T, int E, int S) {
  RouterLayout r;
  // chunks small enough to spread a few thousand rows over the SMs twice, and few enough that the second launch has little to
  // add; their number is part of the order in which a device adds
  const int want = 2 * device_sm_count();
  const int per = (int)(((int64_t)T + want - 1) / want);
  r.rows = std::min(std::max((per + 7) / 8 * 8, 8), 128);
  r.chunks = (T + r.rows - 1) / r.rows;
  r.slots = (int64_t)r.chunks + S;
  auto pad = [](int64_t b) { return (b + 255) / 256 * 256; };
  r.off_c = pad(r.slots * E * 4);
  r.off_z = r.off_c + pad(r.slots * E * 4);
  r.off_n = r.off_z + pad(r.slots * 4);
  r.off_seq = r.off_n + pad(r.slots * 4);
  r.off_ticket = r.off_seq + pad((int64_t)S * ((E + kJoinCols - 1) / kJoinCols) * 12);
  r.bytes = r.off_ticket + 256;
  return r;
}

template <typename T>
int launch_router_fwd_t(const RouterParams& p, cudaStream_t st) {
  void (*k)(RouterParams) = p.E <= 8     ? router_forward_kernel<T, 8, 1>
                            : p.E <= 16  ? router_forward_kernel<T, 16, 1>
                            : p.E <= 32  ? router_forward_kernel<T, 32, 1>
                            : p.E <= 64  ? router_forward_kernel<T, 32, 2>
                            : p.E <= 128 ? router_forward_kernel<T, 32, 4>
                            : p.E <= 256 ? router_forward_kernel<T, 32, 8>
                            : p.E <= 512 ? router_forward_kernel<T, 32, 16>
                                         : router_forward_kernel<T, 32, 32>;
  const int chunks = (p.T + p.rows - 1) / p.rows;
  B200_CHECK_CUDA(launch_chained(k, dim3(chunks), dim3(kRouterThreads), (size_t)(kRouterWarps + 1) * p.E * 4, st, p));
  return 0;
}
template <typename T>
int launch_router_bwd_t(const RouterBwdParams& p, cudaStream_t st) {
  void (*k)(RouterBwdParams) = p.E <= 8     ? router_backward_kernel<T, 8, 1>
                               : p.E <= 16  ? router_backward_kernel<T, 16, 1>
                               : p.E <= 32  ? router_backward_kernel<T, 32, 1>
                               : p.E <= 64  ? router_backward_kernel<T, 32, 2>
                               : p.E <= 128 ? router_backward_kernel<T, 32, 4>
                               : p.E <= 256 ? router_backward_kernel<T, 32, 8>
                               : p.E <= 512 ? router_backward_kernel<T, 32, 16>
                                            : router_backward_kernel<T, 32, 32>;
  const int rows_per_cta = kRouterWarps * (p.E <= 8 ? 4 : p.E <= 16 ? 2 : 1);
  const int grid = std::min((p.T + rows_per_cta - 1) / rows_per_cta, device_sm_count() * 8);
  B200_CHECK_CUDA(launch_chained(k, dim3(grid), dim3(kRouterThreads), 0, st, p));
  return 0;
}

int check_router(int T, int E, int K, int S, int dtype, int scoring, int64_t stride) {
  B200_CHECK_ARG(T >= 0 && T < (1 << 30), "router: T=%d", T);
  B200_CHECK_ARG(E >= 1 && E <= kMaxExperts && K >= 1 && K <= E && K <= kMaxRouterTopk, "router: E=%d K=%d (E up to %d, K up to %d)",
                 E, K, kMaxExperts, kMaxRouterTopk);
  B200_CHECK_ARG(S >= 1 && S < (1 << 20), "router: %d sequences", S);
  B200_CHECK_ARG(dtype >= B200MOE_T_BF16 && dtype <= B200MOE_T_FP32, "router: dtype %d unknown", dtype);
  B200_CHECK_ARG(scoring == 0 || scoring == 1, "router: scoring=%d (0 softmax, 1 sigmoid)", scoring);
  B200_CHECK_ARG(stride >= 0, "router: row stride %lld", (long long)stride);
  return 0;
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" {

int b200moe_router_workspace(int32_t T, int32_t E, int32_t sequences, int64_t* bytes) {
  B200_CHECK_ARG(bytes != nullptr && T >= 0 && E >= 1 && E <= kMaxExperts && sequences >= 1, "router_workspace: T=%d E=%d S=%d", T, E,
                 sequences);
  *bytes = router_layout(T, E, sequences).bytes;
  return 0;
}

int b200moe_router_forward(const void* logits, int64_t stride, int32_t T, int32_t E, int32_t K, int32_t dtype, int32_t scoring,
                           int32_t renormalize, const void* token_mask, const int32_t* cu_seqlens, int32_t sequences,
                           float* topk_weight, int32_t* topk_ids, int32_t* counts, float* balance_loss, float* z_loss, float* lse,
                           int32_t* seg, float* coef, float* stats, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_router(T, E, K, sequences, dtype, scoring, stride)) return rc;
  B200_CHECK_ARG(cu_seqlens != nullptr || sequences == 1, "router: %d sequences without cu_seqlens", sequences);
  B200_CHECK_ARG(counts && balance_loss && z_loss && (T == 0 || (logits && topk_weight && topk_ids)), "router: NULL pointer");
  B200_CHECK_ARG((coef != nullptr) == (stats != nullptr) &&
                     (T == 0 || ((lse != nullptr) == (seg != nullptr) && (lse != nullptr) == (coef != nullptr))),
                 "router: lse, seg, coef and stats go together");
  const RouterLayout r = router_layout(T, E, sequences);
  B200_CHECK_ARG(workspace != nullptr && workspace_bytes >= r.bytes && ((uintptr_t)workspace & 15) == 0,
                 "router: workspace holds %lld bytes of %lld", (long long)workspace_bytes, (long long)r.bytes);
  uint8_t* w = (uint8_t*)workspace;
  cudaStream_t st = (cudaStream_t)stream;
  RouterParams p = {logits, stride, (const uint8_t*)token_mask, cu_seqlens, topk_weight, topk_ids, lse, seg, (float*)w,
                    (int32_t*)(w + r.off_c), (float*)(w + r.off_z), (int32_t*)(w + r.off_n), (int32_t*)(w + r.off_ticket),
                    T, E, K, sequences, r.rows, scoring, renormalize != 0};
  if (T == 0) {
    B200_CHECK_CUDA(cudaMemsetAsync(p.ticket, 0, 4, st));
  } else {
    int rc = dtype == B200MOE_T_BF16   ? launch_router_fwd_t<__nv_bfloat16>(p, st)
             : dtype == B200MOE_T_FP16 ? launch_router_fwd_t<__half>(p, st) : launch_router_fwd_t<float>(p, st);
    if (rc) return rc;
  }
  RouterJoinParams j = {cu_seqlens, p.part_p, p.part_c, p.part_z, p.part_n, p.ticket, counts, coef, (float*)(w + r.off_seq), stats,
                        balance_loss, z_loss, T, E, K, sequences, r.rows, r.chunks};
  B200_CHECK_CUDA(launch_chained(router_join_kernel, dim3(sequences, (E + kJoinCols - 1) / kJoinCols), dim3(kJoinThreads), 0, st, j));
  return 0;
}

int b200moe_router_backward(const void* logits, int64_t stride, int32_t T, int32_t E, int32_t K, int32_t dtype, int32_t scoring,
                            int32_t renormalize, const float* lse, const int32_t* seg, const float* coef, const float* stats,
                            const int32_t* topk_ids, const float* topk_weight, const float* dweight, const float* dbalance,
                            const float* dz, void* dlogits, void* stream) {
  if (int rc = check_router(T, E, K, 1, dtype, scoring, stride)) return rc;
  if (T == 0) return 0;
  B200_CHECK_ARG(logits && lse && seg && coef && stats && topk_ids && topk_weight && dlogits, "router_backward: NULL pointer");
  RouterBwdParams p = {logits, stride, lse, seg, topk_ids, topk_weight, coef, stats, dweight, dbalance, dz, dlogits,
                       T, E, K, scoring, renormalize != 0};
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == B200MOE_T_BF16 ? launch_router_bwd_t<__nv_bfloat16>(p, st)
         : dtype == B200MOE_T_FP16 ? launch_router_bwd_t<__half>(p, st) : launch_router_bwd_t<float>(p, st);
}

}  // extern "C"
