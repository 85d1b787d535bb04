// RMS norms after and before a block, with the branch's gate and the residual's scale, and the 8-bit token quantiser:
//   u = y * rstd(y) * w   (or y, without w)        rstd(v) = 1 / sqrt(mean(v^2) + eps)
//   h = alpha * r + g u                              g: none, or one value per channel, per token or per element
//   n = h * rstd(h) * w'                             stored in the rows' type or as 8-bit integers with the row's scale
// All of it in 32 bits from the inputs, rounded once where it is stored: n is the norm of the unrounded h.
//
// Bound by memory: forward reads y and r and writes h and n (8 bytes a value in 16-bit types), backward reads
// y, r, dh, dn and writes dy and dr (12 bytes).  The threads that share a row take the same columns of every row, in
// 16-byte pieces, so every value is read and written once and the sums over tokens stay with the thread.
// Two forms.  Plain: a row goes straight to registers; any alignment, and the better one for narrow rows.  Ring: a
// thread copies its pieces of the next rows to shared memory while it works on the present one (it reads nothing but
// its own copies, so no barrier), which keeps tens of KB in flight per SM where the plain form waits at every row.
// Wide rows do not fit the plain form's registers: it spills 0.1 KB a thread forward (1025 to 4096 values off the 16-byte grid) and
// 0.2 to 1.2 KB backward (from 4097 values on: off the grid, of two weight types, or too wide for the ring).  4096 x 4099: 406 us
// forward, 1084 us with the backward; 4096 x 7168 of two weight types 94 and 261 us, where one type takes 44 and 125 us in the
// ring; 2048 x 16384 52 us (ring) and 357 us.
// On a B200 (6.55 TB/s measured): forward 8192 x 2880 33 us, 5.7 TB/s; 8192 x 4096 43 us, 6.2 TB/s; 4096 x 7168 45 us,
// 5.3 TB/s.  Backward 4096 x 7168 80 us, 4.4 TB/s; 8192 x 4096 80-84 us, 4.8 TB/s; 16384 x 2048 83 us, 4.8 TB/s: the three
// sums of a row end in a barrier that a CTA's warps reach together.  Quantiser 16384 x 4096 48 us, 4.1 TB/s: a row's reduction
// and scale cost each warp as much as 9 of its values.
#include <algorithm>

#include "rowwise.cuh"

namespace b200moe {

namespace {

constexpr int kRowThreads = 512;          // threads of a CTA at most
constexpr int kMaxNormWidth = 16384;
constexpr int kRingLimit = 224 * 1024;    // shared memory of a ring: what an SM has, less the reductions' slots
template <typename T> constexpr int kMaxPieces = kMaxNormWidth / (16 / (int)sizeof(T)) / kRowThreads;   // 16-byte pieces of a thread

struct NormParams {
  const void* y; const void* r; const void* w; const void* gate; const void* wn;
  int64_t y_stride, r_stride, gate_stride;
  void* h; void* n; int8_t* q; float* q_scale; float* rstd;   // rstd: [2, T], of y and of h; or null
  int T, H, gate_kind, w_f32, gate_f32, wn_f32;
  float alpha, eps;
};

struct NormBwdParams {
  NormParams f;
  const void* dh; const void* dn;
  void* dy; void* dr; void* dgate;    // dgate of kinds token and full; kind channel goes to the partial sums
  float* part;                        // [rows of partial sums][3][H]: dw, dwn, dgate per channel
  int want_dw, want_dwn, want_dgc;
};

template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(kRowThreads, (VEC * NV <= 8) ? 2 : 1)
block_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ float slots[2 * 3 * kMaxRowWarps];
  grid_dep_wait();
  grid_dep_launch();
  RowReduce red(slots);
  const int H = p.H;
  const float inv_h = 1.f / (float)H;
  for (int64_t t0 = (int64_t)blockIdx.x * blockDim.y; t0 < p.T; t0 += (int64_t)gridDim.x * blockDim.y) {
    const int64_t t = t0 + threadIdx.y;
    const bool row = t < p.T;
    float u[NV][VEC], h[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ((int)threadIdx.x + i * (int)blockDim.x) * VEC;
      const bool in = row && c < H;
#pragma unroll
      for (int j = 0; j < VEC; ++j) u[i][j] = h[i][j] = 0.f;
      if (in) load_f<T, VEC>(static_cast<const T*>(p.y) + t * p.y_stride + c, u[i]);
      if (in && p.r != nullptr) load_f<T, VEC>(static_cast<const T*>(p.r) + t * p.r_stride + c, h[i]);
    }
    if (p.w != nullptr) {
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[0] = fmaf(u[i][j], u[i][j], s[0]);
      red.sum(s);
      const float rs = __frsqrt_rn(s[0] * inv_h + p.eps);
      if (row && threadIdx.x == 0 && p.rstd != nullptr) p.rstd[t] = rs;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = ((int)threadIdx.x + i * (int)blockDim.x) * VEC;
        if (c < H) {
          float w[VEC];
          load_param<T, VEC>(p.w, p.w_f32, c, w);
#pragma unroll
          for (int j = 0; j < VEC; ++j) u[i][j] = u[i][j] * rs * w[j];
        }
      }
    }
    float gt = 1.f;
    if (p.gate_kind == B200MOE_GATE_TOKEN && row) {
      float g1[1];
      load_param<T, 1>(p.gate, p.gate_f32, t * p.gate_stride, g1);
      gt = g1[0];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ((int)threadIdx.x + i * (int)blockDim.x) * VEC;
      if (row && c < H) {
        if (p.gate_kind >= B200MOE_GATE_CHANNEL && p.gate_kind != B200MOE_GATE_TOKEN) {
          float g[VEC];
          load_param<T, VEC>(p.gate, p.gate_f32, (p.gate_kind == B200MOE_GATE_FULL ? t * p.gate_stride : 0) + c, g);
#pragma unroll
          for (int j = 0; j < VEC; ++j) u[i][j] *= g[j];
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[i][j] = fmaf(p.alpha, h[i][j], gt * u[i][j]);
        if (p.h != nullptr) store_f<T, VEC>(static_cast<T*>(p.h) + t * H + c, h[i]);
      }
    }
    if (p.wn != nullptr) {
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[0] = fmaf(h[i][j], h[i][j], s[0]);
      red.sum(s);
      const float rs = __frsqrt_rn(s[0] * inv_h + p.eps);
      if (row && threadIdx.x == 0 && p.rstd != nullptr) p.rstd[p.T + t] = rs;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = ((int)threadIdx.x + i * (int)blockDim.x) * VEC;
        if (row && c < H) {
          float w[VEC];
          load_param<T, VEC>(p.wn, p.wn_f32, c, w);
#pragma unroll
          for (int j = 0; j < VEC; ++j) h[i][j] = h[i][j] * rs * w[j];
          if (p.n != nullptr) store_f<T, VEC>(static_cast<T*>(p.n) + t * H + c, h[i]);
        }
      }
    }
    if (p.q != nullptr) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) m = max(m, __float_as_uint(h[i][j]) & 0x7fffffffu);
      m = red.max_u32(m);
      const float s = int8_scale(m);
      const bool bad = m >= 0x7f800000u;
      const float inv = __frcp_rn(s);
      if (row && threadIdx.x == 0) p.q_scale[t] = s;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = ((int)threadIdx.x + i * (int)blockDim.x) * VEC;
        if (row && c < H) {
          Pack<int8_t, VEC> k;
#pragma unroll
          for (int j = 0; j < VEC; ++j) k.v[j] = bad ? (int8_t)0 : (int8_t)quant_int8(h[i][j], s, inv);
          *reinterpret_cast<Pack<int8_t, VEC>*>(p.q + t * H + c) = k;
        }
      }
    }
  }
}

// piece c of a gate per channel, which is fp32 or of the rows' type whatever the weights are
template <typename T, int N2>
__device__ __forceinline__ void load_gate_piece(const NormParams& p, int c, f32x2 (&o)[N2]) {
  if (p.gate_f32) load_piece<T, float>(p.gate, c, o); else load_piece<T, T>(p.gate, c, o);
}

// a thread's pieces of row t as 8-bit integers, and the row's scale, from the bits of its largest magnitude
template <typename T, int NV, int N2>
__device__ __forceinline__ void store_int8_row(const NormParams& p, int64_t t, uint32_t amax_bits, const f32x2 (&v)[NV][N2], int chunks) {
  constexpr int VEC = 2 * N2;
  const int tid = (int)threadIdx.x, tpr = (int)blockDim.x;
  const float s = int8_scale(amax_bits), inv = __fdividef(1.f, s);       // (quant_int8 needs no exact reciprocal)
  const bool bad = amax_bits >= 0x7f800000u;
  if (tid == 0) p.q_scale[t] = s;
  uint8_t* out = reinterpret_cast<uint8_t*>(p.q + t * p.H) + tid * VEC;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (tid + i * tpr < chunks) {
      uint32_t k[N2 / 2];
      quant_int8(v[i], s, inv, k);
      if constexpr (N2 == 4) {
        *reinterpret_cast<uint2*>(out + i * tpr * VEC) = bad ? make_uint2(0, 0) : make_uint2(k[0], k[1]);
      } else {
        *reinterpret_cast<uint32_t*>(out + i * tpr * VEC) = bad ? 0u : k[0];
      }
    }
}

// Forward over a ring of two to four rows in shared memory, 16-byte pieces and pairs of values throughout, 16 values to a thread.
// GATE: 0 none or per token, 1 per channel, 2 per element.  P: type of the norms' weights.
// HOLD: the weights (times the gate per channel) stay in registers over the rows.  L1 would serve them at every row, which
// costs it as much as the rows themselves (66 % of its data pipe with fp32 weights; 43.8 -> 36.8 us at 8192 x 2880).  It takes
// 85 registers, so 768 threads an SM; rows so wide that only one CTA of those would fit read the weights again and have two
// CTAs of 64 registers (4096 x 7168: 47 against 65 us).
constexpr int kNormValues = 16;
constexpr int kHoldThreads = 768, kNoHoldThreads = 1024;      // of an SM
template <typename T, typename P, bool POST, int GATE, bool HOLD>
__global__ void __launch_bounds__(HOLD ? kHoldThreads : kNoHoldThreads, 1)
block_norm_ring_kernel(const __grid_constant__ NormParams p, int stages) {
  constexpr int VEC = 16 / sizeof(T), NV = kNormValues / VEC, N2 = VEC / 2;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(16) float slots[2 * 32 * 4];
  CtaReduce red(slots);
  grid_dep_wait();
  grid_dep_launch();
  const int chunks = p.H / VEC, tpr = (int)blockDim.x, tid = (int)threadIdx.x;
  const bool res = p.r != nullptr, next = p.wn != nullptr;
  const uint32_t array_bytes = (uint32_t)chunks * 16;
  const uint32_t at_g = array_bytes * (1 + res), stage_bytes = at_g + (GATE == 2 ? array_bytes : 0);
  const uint32_t mine = smem_u32(ring) + (uint32_t)tid * 16;
  const float inv_h = 1.f / (float)p.H;
  auto fetch = [&](int64_t t, uint32_t at) {
    if (t < p.T) {
      const uint4* y = reinterpret_cast<const uint4*>(static_cast<const T*>(p.y) + t * p.y_stride) + tid;
      const uint4* r = reinterpret_cast<const uint4*>(static_cast<const T*>(p.r) + t * p.r_stride) + tid;
      const uint4* g = reinterpret_cast<const uint4*>(static_cast<const T*>(p.gate) + t * p.gate_stride) + tid;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (tid + i * tpr < chunks) {
          const uint32_t dst = at + (uint32_t)(i * tpr) * 16;
          copy16_async(dst, y + i * tpr);
          if (res) copy16_async(dst + array_bytes, r + i * tpr);
          if (GATE == 2) copy16_async(dst + at_g, g + i * tpr);
        }
      }
    }
    copy_commit();
  };
  // the factor of y in piece c that the rows share, and the next norm's weights
  auto load_factor = [&](int c, f32x2 (&f)[N2]) {
#pragma unroll
    for (int j = 0; j < N2; ++j) f[j] = both(1.f);
    if (POST) load_piece<T, P>(p.w, c, f);
    if (GATE == 1) {
      f32x2 g[N2];
      load_gate_piece<T>(p, c, g);
#pragma unroll
      for (int j = 0; j < N2; ++j) f[j] = mul2(f[j], g[j]);
    }
  };
  const int64_t step = gridDim.x;
  const uint32_t end = mine + stages * stage_bytes;
  uint32_t at = mine, other = mine;               // the present row, and the stage that the row before has left
  for (int s = 0; s < stages - 1; ++s, other += stage_bytes) fetch(blockIdx.x + s * step, other);
  f32x2 hold_f[HOLD ? NV : 1][N2], hold_n[HOLD ? NV : 1][N2];
  if (HOLD) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * tpr < chunks) {
        load_factor(tid + i * tpr, hold_f[i]);
        if (next) load_piece<T, P>(p.wn, tid + i * tpr, hold_n[i]);
      }
  }
  const bool token = GATE == 0 && p.gate_kind == B200MOE_GATE_TOKEN;
  auto token_gate = [&](int64_t t) {
    float g[1] = {1.f};
    if (token && t < p.T) load_param<T, 1>(p.gate, p.gate_f32, t * p.gate_stride, g);
    return g[0];
  };
  float next_gate = token_gate(blockIdx.x);       // a row ahead, as the rows themselves
  for (int64_t t = blockIdx.x; t < p.T; t += step) {
    if (stages == 2) copy_wait<0>(); else if (stages == 3) copy_wait<1>(); else copy_wait<2>();
    fetch(t + (stages - 1) * step, other);
    f32x2 h[NV][N2];
    float scale = 1.f;                            // rstd(y) and a token's gate
    const float gt = next_gate;
    next_gate = token_gate(t + step);
    if (POST) {
      f32x2 ss = both(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (tid + i * tpr < chunks) {
          unpack16(lds16(at + (uint32_t)(i * tpr) * 16), h[i], T());
#pragma unroll
          for (int j = 0; j < N2; ++j) ss = fma2(h[i][j], h[i][j], ss);
        }
      const float sum = red.sum(both_of(ss));
      scale = rsqrtf(sum * inv_h + p.eps);
      if (tid == 0 && p.rstd != nullptr) p.rstd[t] = scale;
    }
    if (GATE == 0) scale *= gt;
    const f32x2 scale2 = both(scale), alpha2 = both(p.alpha);
    f32x2 ss = both(0.f);
    uint4* ho = reinterpret_cast<uint4*>(static_cast<T*>(p.h) + t * p.H) + tid;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * tpr < chunks) {
        const uint32_t src = at + (uint32_t)(i * tpr) * 16;
        f32x2 f[N2], r[N2];
        if (!POST) unpack16(lds16(src), h[i], T());
        if (HOLD) {
#pragma unroll
          for (int j = 0; j < N2; ++j) f[j] = hold_f[i][j];
        } else {
          load_factor(tid + i * tpr, f);
        }
#pragma unroll
        for (int j = 0; j < N2; ++j) h[i][j] = mul2(h[i][j], (POST || GATE == 1) ? mul2(f[j], scale2) : scale2);
        if (GATE == 2) {
          unpack16(lds16(src + at_g), r, T());
#pragma unroll
          for (int j = 0; j < N2; ++j) h[i][j] = mul2(h[i][j], r[j]);
        }
        if (res) {
          unpack16(lds16(src + array_bytes), r, T());
#pragma unroll
          for (int j = 0; j < N2; ++j) h[i][j] = fma2(r[j], alpha2, h[i][j]);
        }
#pragma unroll
        for (int j = 0; j < N2; ++j) ss = fma2(h[i][j], h[i][j], ss);
        if (p.h != nullptr) ho[i * tpr] = pack16(h[i], T());
      }
    if (next) {
      const float sum = red.sum(both_of(ss));
      const float rh = rsqrtf(sum * inv_h + p.eps);
      if (tid == 0 && p.rstd != nullptr) p.rstd[p.T + t] = rh;
      const f32x2 rh2 = both(rh);
      uint4* no = reinterpret_cast<uint4*>(static_cast<T*>(p.n) + t * p.H) + tid;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (tid + i * tpr < chunks) {
          f32x2 f[N2];
          if (HOLD) {
#pragma unroll
            for (int j = 0; j < N2; ++j) f[j] = hold_n[i][j];
          } else {
            load_piece<T, P>(p.wn, tid + i * tpr, f);
          }
#pragma unroll
          for (int j = 0; j < N2; ++j) h[i][j] = mul2(h[i][j], mul2(f[j], rh2));
          if (p.n != nullptr) no[i * tpr] = pack16(h[i], T());
        }
    }
    if (p.q != nullptr) {
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (tid + i * tpr < chunks) amax = max_abs_nan(amax, h[i]);
      const uint32_t m = red.max_u32(__float_as_uint(amax) & 0x7fffffffu);
      store_int8_row<T>(p, t, m, h, chunks);
    }
    at = at + stage_bytes == end ? mine : at + stage_bytes;
    other = other + stage_bytes == end ? mine : other + stage_bytes;
  }
}

// The token quantiser by itself over the same ring: no norm in between, so 32 values to a thread, which halves what a row
// costs whatever its width (reduction, scale, copies).
constexpr int kQuantValues = 32, kQuantThreads = 768;      // of an SM
template <typename T>
__global__ void __launch_bounds__(kRowThreads, 1)
quant_ring_kernel(const __grid_constant__ NormParams p, int stages) {
  constexpr int VEC = 16 / sizeof(T), NV = kQuantValues / VEC, N2 = VEC / 2;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(16) float slots[2 * 32 * 4];
  CtaReduce red(slots);
  grid_dep_wait();
  grid_dep_launch();
  const int chunks = p.H / VEC, tpr = (int)blockDim.x, tid = (int)threadIdx.x;
  const uint32_t stage_bytes = (uint32_t)chunks * 16;
  const uint32_t mine = smem_u32(ring) + (uint32_t)tid * 16, end = mine + stages * stage_bytes;
  auto fetch = [&](int64_t t, uint32_t at) {
    if (t < p.T) {
      const uint4* y = reinterpret_cast<const uint4*>(static_cast<const T*>(p.y) + t * p.y_stride) + tid;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (tid + i * tpr < chunks) copy16_async(at + (uint32_t)(i * tpr) * 16, y + i * tpr);
    }
    copy_commit();
  };
  const int64_t step = gridDim.x;
  uint32_t at = mine, other = mine;
  for (int s = 0; s < stages - 1; ++s, other += stage_bytes) fetch(blockIdx.x + s * step, other);
  for (int64_t t = blockIdx.x; t < p.T; t += step) {
    if (stages == 2) copy_wait<0>(); else if (stages == 3) copy_wait<1>(); else copy_wait<2>();
    fetch(t + (stages - 1) * step, other);
    f32x2 v[NV][N2];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * tpr < chunks) {
        unpack16(lds16(at + (uint32_t)(i * tpr) * 16), v[i], T());
        amax = max_abs_nan(amax, v[i]);
      }
    const uint32_t m = red.max_u32(__float_as_uint(amax) & 0x7fffffffu);
    store_int8_row<T>(p, t, m, v, chunks);
    at = at + stage_bytes == end ? mine : at + stage_bytes;
    other = other + stage_bytes == end ? mine : other + stage_bytes;
  }
}

// Backward.  With k = h rstd(h), e = dh + rstd(h) w' dn and c = rstd(h) mean(w' dn k) the gradient that reaches h is e - c k, and
// the sum that the norm of y needs, S = sum(w y g (e - c k)), is A - c B with A = sum(w y g e), B = sum(w y g k): all three sums
// of a row are formed in one reduction.  A gate per token is a factor of A and B, and its own gradient is rstd(y)(A - cB).
// The part of dy along y is (y rstd(y)) (rstd(y) (rstd(y) S) / H).  No power of rstd is formed: its cube leaves the
// 32-bit range where a row's RMS passes 5e12, while the row's sum of squares stays in it up to an RMS of 1.8e19 / sqrt(H).
// The gradients of the weights and of a gate per channel are summed over the CTA's rows in registers, stored once per
// CTA and joined by column_sum_kernel in a fixed order: no atomics, the same bits on every run.
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(kRowThreads, 1)
block_norm_bwd_kernel(const __grid_constant__ NormBwdParams b) {
  __shared__ float slots[2 * 3 * kMaxRowWarps];
  grid_dep_wait();
  grid_dep_launch();
  const NormParams& p = b.f;
  RowReduce red(slots);
  const int H = p.H;
  const float inv_h = 1.f / (float)H;
  const bool by_value = p.gate_kind == B200MOE_GATE_CHANNEL || p.gate_kind == B200MOE_GATE_FULL;
  float aw[NV][VEC], an[NV][VEC], ag[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) aw[i][j] = an[i][j] = ag[i][j] = 0.f;
  for (int64_t t0 = (int64_t)blockIdx.x * blockDim.y; t0 < p.T; t0 += (int64_t)gridDim.x * blockDim.y) {
    const int64_t t = t0 + threadIdx.y;
    const bool row = t < p.T;
    float gt = 1.f, ry = 1.f, rh = 0.f;
    if (row) {
      if (p.gate_kind == B200MOE_GATE_TOKEN) {
        float g1[1];
        load_param<T, 1>(p.gate, p.gate_f32, t * p.gate_stride, g1);
        gt = g1[0];
      }
      if (p.w != nullptr) ry = p.rstd[t];
      if (p.wn != nullptr) rh = p.rstd[p.T + t];
    }
    const float yg = ry * gt, alpha_h = p.alpha * rh;
    float y[NV][VEC], h[NV][VEC], e[NV][VEC], dn[NV][VEC];
    float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ((int)threadIdx.x + i * (int)blockDim.x) * VEC;
      const bool in = row && c < H;
#pragma unroll
      for (int j = 0; j < VEC; ++j) y[i][j] = h[i][j] = e[i][j] = dn[i][j] = 0.f;
      if (in) {
        load_f<T, VEC>(static_cast<const T*>(p.y) + t * p.y_stride + c, y[i]);
        if (p.r != nullptr) load_f<T, VEC>(static_cast<const T*>(p.r) + t * p.r_stride + c, h[i]);
        if (b.dh != nullptr) load_f<T, VEC>(static_cast<const T*>(b.dh) + t * H + c, e[i]);
        if (b.dn != nullptr) load_f<T, VEC>(static_cast<const T*>(b.dn) + t * H + c, dn[i]);
        float g[VEC], w[VEC], wn[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) { g[j] = gt; w[j] = 1.f; wn[j] = 0.f; }
        if (by_value) load_param<T, VEC>(p.gate, p.gate_f32, (p.gate_kind == B200MOE_GATE_FULL ? t * p.gate_stride : 0) + c, g);
        if (p.w != nullptr) load_param<T, VEC>(p.w, p.w_f32, c, w);
        if (p.wn != nullptr) load_param<T, VEC>(p.wn, p.wn_f32, c, wn);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float v = by_value ? y[i][j] * w[j] * g[j] : y[i][j] * w[j];
          h[i][j] = fmaf(alpha_h, h[i][j], v * yg * rh);          // h rstd(h)
          const float wd = wn[j] * dn[i][j];
          e[i][j] = fmaf(rh, wd, e[i][j]);
          s[0] = fmaf(wd, h[i][j], s[0]);
          s[1] = fmaf(v, e[i][j], s[1]);
          s[2] = fmaf(v, h[i][j], s[2]);
        }
      }
    }
    red.sum(s);
    const float c1 = rh * s[0] * inv_h;
    const float sum_y = ry * (s[1] - c1 * s[2]);
    const float cy = (p.w != nullptr) ? yg * sum_y * inv_h : 0.f;
    if (row && threadIdx.x == 0 && p.gate_kind == B200MOE_GATE_TOKEN && b.dgate != nullptr) {
      const float one[1] = {sum_y};
      store_param<T, 1>(b.dgate, p.gate_f32, t, one);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ((int)threadIdx.x + i * (int)blockDim.x) * VEC;
      if (row && c < H) {
        float g[VEC], w[VEC], out[VEC], dr[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) { g[j] = gt; w[j] = 1.f; }
        if (by_value) load_param<T, VEC>(p.gate, p.gate_f32, (p.gate_kind == B200MOE_GATE_FULL ? t * p.gate_stride : 0) + c, g);
        if (p.w != nullptr) load_param<T, VEC>(p.w, p.w_f32, c, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = fmaf(-c1, h[i][j], e[i][j]);
          dr[j] = p.alpha * d;
          const float du = d * g[j], yr = y[i][j] * ry;
          out[j] = fmaf(ry * w[j], du, -cy * yr);
          aw[i][j] = fmaf(du, yr, aw[i][j]);
          an[i][j] = fmaf(dn[i][j], h[i][j], an[i][j]);
          const float dg = d * (yr * w[j]);
          ag[i][j] += dg;
          g[j] = dg;
        }
        if (b.dy != nullptr) store_f<T, VEC>(static_cast<T*>(b.dy) + t * H + c, out);
        if (b.dr != nullptr) store_f<T, VEC>(static_cast<T*>(b.dr) + t * H + c, dr);
        if (p.gate_kind == B200MOE_GATE_FULL && b.dgate != nullptr) store_param<T, VEC>(b.dgate, p.gate_f32, t * H + c, g);
      }
    }
  }
  if (b.part != nullptr) {
    float* o = b.part + ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * 3 * H;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ((int)threadIdx.x + i * (int)blockDim.x) * VEC;
      if (c < H) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (b.want_dw) o[c + j] = aw[i][j];
          if (b.want_dwn) o[H + c + j] = an[i][j];
          if (b.want_dgc) o[2 * H + c + j] = ag[i][j];
        }
      }
    }
  }
}

// Backward over a ring of rows in shared memory.  What a row needs twice (y, dn) is read from there again instead of held,
// so that a thread's values and their sums over tokens fit the registers.  GATE and P as in the forward kernel.
// VALUES of a row to a thread: 16, and where two CTAs of those would not fit an SM (rows of more than 4096 values), 8 in up
// to 896 threads, since the one CTA's phases between its barriers need the warps (4096 x 7168: 79 against 88 us; a gate's
// values and their sums do not fit there).  Weights held in registers cost more in occupancy than their loads do
// (8192 x 4096: 90 against 80 us).
// 896 threads leave 72 registers, which the form with both norms takes; at 1024 threads it spills with fp32 weights.
constexpr int kWideThreads = 896;
template <typename T, typename P, int GATE, bool POST, bool NEXT, int VALUES>
__global__ void __launch_bounds__(VALUES == 8 ? kWideThreads : kRowThreads, 1)
block_norm_bwd_ring_kernel(const __grid_constant__ NormBwdParams b) {
  constexpr int VEC = 16 / sizeof(T), NV = VALUES / VEC, N2 = VEC / 2;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(16) float slots[2 * 32 * 4];
  const NormParams& p = b.f;
  CtaReduce red(slots);
  grid_dep_wait();
  grid_dep_launch();
  const int chunks = p.H / VEC, tpr = (int)blockDim.x, tid = (int)threadIdx.x;
  const bool res = NEXT && p.r != nullptr, has_dh = b.dh != nullptr, has_dn = NEXT && b.dn != nullptr;   // (h is needed with NEXT only)
  const uint32_t array_bytes = (uint32_t)chunks * 16;
  const uint32_t at_r = array_bytes, at_h = at_r + (res ? array_bytes : 0), at_n = at_h + (has_dh ? array_bytes : 0);
  const uint32_t at_g = at_n + (has_dn ? array_bytes : 0), stage_bytes = at_g + (GATE == 2 ? array_bytes : 0);
  const uint32_t mine = smem_u32(ring) + (uint32_t)tid * 16;
  const float inv_h = 1.f / (float)p.H;
  const bool token = GATE == 0 && p.gate_kind == B200MOE_GATE_TOKEN;
  auto fetch = [&](int64_t t, uint32_t at) {
    if (t < p.T) {
      const uint4* y = reinterpret_cast<const uint4*>(static_cast<const T*>(p.y) + t * p.y_stride) + tid;
      const uint4* r = reinterpret_cast<const uint4*>(static_cast<const T*>(p.r) + t * p.r_stride) + tid;
      const uint4* dh = reinterpret_cast<const uint4*>(static_cast<const T*>(b.dh) + t * p.H) + tid;
      const uint4* dn = reinterpret_cast<const uint4*>(static_cast<const T*>(b.dn) + t * p.H) + tid;
      const uint4* g = reinterpret_cast<const uint4*>(static_cast<const T*>(p.gate) + t * p.gate_stride) + tid;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (tid + i * tpr < chunks) {
          const uint32_t dst = at + (uint32_t)(i * tpr) * 16;
          copy16_async(dst, y + i * tpr);
          if (res) copy16_async(dst + at_r, r + i * tpr);
          if (has_dh) copy16_async(dst + at_h, dh + i * tpr);
          if (has_dn) copy16_async(dst + at_n, dn + i * tpr);
          if (GATE == 2) copy16_async(dst + at_g, g + i * tpr);
        }
      }
    }
    copy_commit();
  };
  f32x2 aw[POST ? NV : 1][N2], an[NEXT ? NV : 1][N2], ag[GATE == 1 ? NV : 1][N2];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < N2; ++j) {
      if (POST) aw[i][j] = both(0.f);
      if (NEXT) an[i][j] = both(0.f);
      if (GATE == 1) ag[i][j] = both(0.f);
    }
  const int64_t step = gridDim.x;
  fetch(blockIdx.x, mine);
  // a row's scalars come a row ahead, as the rows themselves: a load in front of the sums would cost every row its latency
  struct RowScalars {
    float ry, rh, gt;
  };
  auto scalars = [&](int64_t t) {
    RowScalars r = {1.f, 0.f, 1.f};
    if (t < p.T) {
      if (POST) r.ry = p.rstd[t];
      if (NEXT) r.rh = p.rstd[p.T + t];
      if (token) {
        float g[1];
        load_param<T, 1>(p.gate, p.gate_f32, t * p.gate_stride, g);
        r.gt = g[0];
      }
    }
    return r;
  };
  RowScalars ahead = scalars(blockIdx.x);
  uint32_t at = mine, other = mine + stage_bytes;
  for (int64_t t = blockIdx.x; t < p.T; t += step) {
    copy_wait<0>();
    fetch(t + step, other);                       // the stage that the row before has left
    const float ry = ahead.ry, rh = ahead.rh, gt = ahead.gt;
    ahead = scalars(t + step);
    // h is carried as h rstd(h), the form in which the weights' sum and the correction along h take it
    const f32x2 rh2 = both(rh), alpha_h = both(p.alpha * rh), yg_h = both(ry * gt * rh);
    f32x2 h[NEXT ? NV : 1][N2], e[NV][N2];
    f32x2 s0 = both(0.f), s1 = both(0.f), s2 = both(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * tpr < chunks) {
        const uint32_t src = at + (uint32_t)(i * tpr) * 16;
        f32x2 v[N2], f[N2];
        // v = w y (g): what the norm's sum takes the gradient times
        unpack16(lds16(src), v, T());
        if (POST) {
          load_piece<T, P>(p.w, tid + i * tpr, f);
#pragma unroll
          for (int j = 0; j < N2; ++j) v[j] = mul2(v[j], f[j]);
        }
        if (GATE != 0) {
          if (GATE == 1) load_gate_piece<T>(p, tid + i * tpr, f); else unpack16(lds16(src + at_g), f, T());
#pragma unroll
          for (int j = 0; j < N2; ++j) v[j] = mul2(v[j], f[j]);
        }
        if (has_dh) {
          unpack16(lds16(src + at_h), e[i], T());
        } else {
#pragma unroll
          for (int j = 0; j < N2; ++j) e[i][j] = both(0.f);
        }
        if (NEXT) {
          if (res) {
            unpack16(lds16(src + at_r), f, T());
#pragma unroll
            for (int j = 0; j < N2; ++j) h[i][j] = fma2(v[j], yg_h, mul2(f[j], alpha_h));
          } else {
#pragma unroll
            for (int j = 0; j < N2; ++j) h[i][j] = mul2(v[j], yg_h);
          }
          if (has_dn) {
            f32x2 d[N2];
            unpack16(lds16(src + at_n), d, T());
            load_piece<T, P>(p.wn, tid + i * tpr, f);
#pragma unroll
            for (int j = 0; j < N2; ++j) {
              an[i][j] = fma2(d[j], h[i][j], an[i][j]);
              d[j] = mul2(d[j], f[j]);
              e[i][j] = fma2(d[j], rh2, e[i][j]);
              s0 = fma2(d[j], h[i][j], s0);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < N2; ++j) {
          s1 = fma2(v[j], e[i][j], s1);
          if (NEXT) s2 = fma2(v[j], h[i][j], s2);
        }
      }
    float t0 = both_of(s0), t1 = both_of(s1), t2 = both_of(s2);
    if (POST || NEXT || token) red.sum3(t0, t1, t2);
    const float c1 = NEXT ? rh * t0 * inv_h : 0.f;
    const float sum_y = ry * (t1 - c1 * t2);
    const float cy = POST ? ry * sum_y * inv_h : 0.f;       // of y rstd(y) gate
    if (token && tid == 0 && b.dgate != nullptr) {
      const float one[1] = {sum_y};
      store_param<T, 1>(b.dgate, p.gate_f32, t, one);
    }
    const f32x2 c2 = both(-c1), cy2 = both(-cy), alpha2 = both(p.alpha), yg2 = both(ry * gt);
    uint4* dyo = reinterpret_cast<uint4*>(static_cast<T*>(b.dy) + t * p.H) + tid;
    uint4* dro = reinterpret_cast<uint4*>(static_cast<T*>(b.dr) + t * p.H) + tid;
    uint4* dgo = reinterpret_cast<uint4*>(static_cast<T*>(b.dgate) + t * p.H) + tid;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * tpr < chunks) {
        const uint32_t src = at + (uint32_t)(i * tpr) * 16;
        f32x2 y[N2], f[N2], d[N2];
#pragma unroll
        for (int j = 0; j < N2; ++j) d[j] = NEXT ? fma2(h[i][j], c2, e[i][j]) : e[i][j];
        if (b.dr != nullptr) {
#pragma unroll
          for (int j = 0; j < N2; ++j) f[j] = mul2(d[j], alpha2);
          dro[i * tpr] = pack16(f, T());
        }
        unpack16(lds16(src), y, T());
        if (POST) load_piece<T, P>(p.w, tid + i * tpr, f);
        if (GATE != 0) {
          f32x2 g[N2], dg[N2];
          if (GATE == 1) load_gate_piece<T>(p, tid + i * tpr, g); else unpack16(lds16(src + at_g), g, T());
#pragma unroll
          for (int j = 0; j < N2; ++j) {
            const f32x2 u = POST ? mul2(mul2(y[j], yg2), f[j]) : y[j];          // (gt is 1 here)
            if (GATE == 1) ag[i][j] = fma2(d[j], u, ag[i][j]); else dg[j] = mul2(d[j], u);
            d[j] = mul2(d[j], g[j]);
          }
          if (GATE == 2 && b.dgate != nullptr) dgo[i * tpr] = pack16(dg, T());
        }
        // d times a token's gate is the gradient of u
        if (POST) {
#pragma unroll
          for (int j = 0; j < N2; ++j) {
            const f32x2 yr = mul2(y[j], yg2);
            aw[i][j] = fma2(d[j], yr, aw[i][j]);
            d[j] = fma2(d[j], mul2(f[j], yg2), mul2(yr, cy2));
          }
        } else if (GATE == 0) {
#pragma unroll
          for (int j = 0; j < N2; ++j) d[j] = mul2(d[j], yg2);
        }
        if (b.dy != nullptr) dyo[i * tpr] = pack16(d, T());
      }
    const uint32_t swap = at;
    at = other;
    other = swap;
  }
  if (b.part != nullptr) {
    f32x2* o = reinterpret_cast<f32x2*>(b.part + (int64_t)blockIdx.x * 3 * p.H);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = tid + i * tpr;
      if (c < chunks) {
#pragma unroll
        for (int j = 0; j < N2; ++j) {
          if (POST && b.want_dw) o[c * N2 + j] = aw[i][j];
          if (NEXT && b.want_dwn) o[p.H / 2 + c * N2 + j] = an[i][j];
          if (GATE == 1 && b.want_dgc) o[p.H + c * N2 + j] = ag[i][j];
        }
      }
    }
  }
}

// dst[c] = sum over the partial rows, in ascending order within 32 interleaved groups that are then added in order.  The
// groups are many because the columns are few: with 8 of them this was most of a backward pass over narrow rows.
struct ColumnSumParams {
  const float* part;
  void* dst[3];
  int f32[3];
  int rows, H;
};
constexpr int kSumGroups = 32;
template <typename T>
__global__ void __launch_bounds__(kSumGroups * 32)
column_sum_kernel(const __grid_constant__ ColumnSumParams p) {
  __shared__ float s[kSumGroups][33];
  grid_dep_wait();
  grid_dep_launch();
  const int which = blockIdx.y, col = blockIdx.x * 32 + (threadIdx.x & 31), grp = threadIdx.x >> 5;
  if (p.dst[which] == nullptr) return;
  float a = 0.f;
  if (col < p.H)
#pragma unroll 8
    for (int r = grp; r < p.rows; r += kSumGroups) a += p.part[((int64_t)r * 3 + which) * p.H + col];
  s[grp][threadIdx.x & 31] = a;
  __syncthreads();
  if (grp == 0 && col < p.H) {
    float v[1] = {0.f};
#pragma unroll
    for (int g = 0; g < kSumGroups; ++g) v[0] += s[g][threadIdx.x];
    store_param<T, 1>(p.dst[which], p.f32[which], col, v);
  }
}

// threads per row and rows per CTA for `chunks` pieces of a row, nv of them to a thread
struct RowShape {
  int nv, tpr, rows;
};
RowShape row_shape(int64_t chunks) {
  RowShape s;
  s.nv = 1;
  while ((chunks + s.nv - 1) / s.nv > kRowThreads) s.nv *= 2;
  s.tpr = (int)round_up64((chunks + s.nv - 1) / s.nv, 32);
  s.rows = std::max(1, 256 / s.tpr);
  return s;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// 16-byte pieces need every row of every tensor to start on a 16-byte boundary
template <typename T>
bool vector_ok(const NormParams& p) {
  constexpr int V = 16 / sizeof(T);
  return p.H % V == 0 && (p.y_stride % V) == 0 && (p.r == nullptr || p.r_stride % V == 0) &&
         (p.gate_kind != B200MOE_GATE_FULL || p.gate_stride % V == 0) && aligned16(p.y) && aligned16(p.r) && aligned16(p.w) &&
         (p.gate_kind == B200MOE_GATE_TOKEN || aligned16(p.gate)) && aligned16(p.wn) && aligned16(p.h) && aligned16(p.n) && aligned16(p.q);
}

// The ring needs its gate rows in the rows' type, its weights in one type, and a width that gives its warps something to do.
// Plain against ring, us (bf16 with a residual and both norms; forward, backward):  4096 x 256: 3.4, 19.0 against 4.3, 17.6;
// 4096 x 512: 6.1, 23.9 against 4.7, 21.3;  128 x 512: 2.7, 7.4 against 2.6, 5.7;  64 x 2880: 2.9, 9.2 against 2.8, 8.6;
// 4096 x 2880: 40.0, 73.2 against 16.9, 41.2.
template <typename T>
bool ring_ok(const NormParams& p, bool vec) {
  return vec && p.H >= 512 && (sizeof(T) == 4 || p.w == nullptr || p.wn == nullptr || p.w_f32 == p.wn_f32) &&
         (p.gate_kind != B200MOE_GATE_FULL || sizeof(T) == 4 || !p.gate_f32);
}
// whether the weights are fp32 (they are of one type)
bool fp32_weights(const NormParams& p) { return (p.w != nullptr && p.w_f32) || (p.wn != nullptr && p.wn_f32); }
int ring_gate(const NormParams& p) {
  return p.gate_kind == B200MOE_GATE_CHANNEL ? 1 : p.gate_kind == B200MOE_GATE_FULL ? 2 : 0;
}
template <typename T, typename P, bool POST, bool HOLD>
void (*fwd_ring_g(int g))(NormParams, int) {
  return g == 0 ? block_norm_ring_kernel<T, P, POST, 0, HOLD> : g == 1 ? block_norm_ring_kernel<T, P, POST, 1, HOLD>
                                                                      : block_norm_ring_kernel<T, P, POST, 2, HOLD>;
}
template <typename T, typename P>
void (*fwd_ring(const NormParams& p, bool hold))(NormParams, int) {
  const int g = ring_gate(p);
  if (p.w != nullptr) return hold ? fwd_ring_g<T, P, true, true>(g) : fwd_ring_g<T, P, true, false>(g);
  return hold ? fwd_ring_g<T, P, false, true>(g) : fwd_ring_g<T, P, false, false>(g);
}
template <typename T, typename P, int GATE, int VALUES>
void (*bwd_ring_g(const NormParams& p))(NormBwdParams) {
  if (p.w != nullptr)
    return p.wn != nullptr ? block_norm_bwd_ring_kernel<T, P, GATE, true, true, VALUES> : block_norm_bwd_ring_kernel<T, P, GATE, true, false, VALUES>;
  return p.wn != nullptr ? block_norm_bwd_ring_kernel<T, P, GATE, false, true, VALUES> : block_norm_bwd_ring_kernel<T, P, GATE, false, false, VALUES>;
}
template <typename T, typename P>
void (*bwd_ring(const NormParams& p, bool wide))(NormBwdParams) {
  const int g = ring_gate(p);
  if (g == 0) return wide ? bwd_ring_g<T, P, 0, 8>(p) : bwd_ring_g<T, P, 0, 16>(p);
  return g == 1 ? bwd_ring_g<T, P, 1, 16>(p) : bwd_ring_g<T, P, 2, 16>(p);
}

template <typename T>
int launch_norm_t(const NormParams& p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = vector_ok<T>(p);
  if (ring_ok<T>(p, vec) && p.r == nullptr && p.w == nullptr && p.wn == nullptr && p.gate_kind == B200MOE_GATE_NONE && p.h == nullptr) {
    constexpr int NV = kQuantValues / V;
    const int tpr = (int)round_up64((p.H / V + NV - 1) / NV, 32), row_bytes = p.H * (int)sizeof(T);
    const int per_sm = std::max(1, std::min(kQuantThreads / tpr, kRingLimit / (2 * row_bytes + 2048)));
    const int ahead = std::min((40 * 1024 + per_sm * row_bytes - 1) / (per_sm * row_bytes), 3);
    const int stages = std::max(2, std::min(ahead + 1, kRingLimit / per_sm / row_bytes));
    const int grid = (int)std::min<int64_t>(p.T, (int64_t)device_sm_count() * per_sm);
    B200_CHECK_CUDA(cudaFuncSetAttribute(quant_ring_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingLimit));
    B200_CHECK_CUDA(launch_chained(quant_ring_kernel<T>, dim3(grid), dim3(tpr), (size_t)stages * row_bytes, st, p, stages));
    return 0;
  }
  if (ring_ok<T>(p, vec)) {
    constexpr int NV = kNormValues / V;
    const int tpr = (int)round_up64((p.H / V + NV - 1) / NV, 32);
    const int arrays = 1 + (p.r != nullptr) + (p.gate_kind == B200MOE_GATE_FULL);
    const int row_bytes = arrays * p.H * (int)sizeof(T);
    if (2 * row_bytes <= kRingLimit && tpr <= kNoHoldThreads) {
      const bool hold = 2 * tpr <= kHoldThreads;
      const int per_sm = std::max(1, std::min((hold ? kHoldThreads : kNoHoldThreads) / tpr, kRingLimit / (2 * row_bytes + 2048)));
      // Rows ahead until an SM has 40 KB on their way, which its share of the memory's rate times the latency asks for
      // (the quantiser at 16384 x 4096, 24 KB with one row ahead).
      const int ahead = std::min((40 * 1024 + per_sm * row_bytes - 1) / (per_sm * row_bytes), 3);
      const int stages = std::max(2, std::min(ahead + 1, kRingLimit / per_sm / row_bytes));
      const size_t smem = (size_t)stages * row_bytes;
      const int grid = (int)std::min<int64_t>(p.T, (int64_t)device_sm_count() * per_sm);
      void (*k)(NormParams, int) = fp32_weights(p) ? fwd_ring<T, float>(p, hold) : fwd_ring<T, T>(p, hold);
      B200_CHECK_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingLimit));
      B200_CHECK_CUDA(launch_chained(k, dim3(grid), dim3(tpr), smem, st, p, stages));
      return 0;
    }
  }
  const RowShape s = row_shape(vec ? p.H / V : p.H);
  const dim3 block(s.tpr, s.rows);
  const int per_sm = std::max(1, ((V * s.nv <= 8) ? 1024 : 512) / (s.tpr * s.rows));
  const int grid = (int)std::min<int64_t>((p.T + s.rows - 1) / s.rows, (int64_t)device_sm_count() * per_sm);
  void (*k)(NormParams) = nullptr;
  if (vec)
    k = s.nv == 1 ? block_norm_kernel<T, V, 1> : s.nv == 2 ? block_norm_kernel<T, V, 2> : s.nv == 4 ? block_norm_kernel<T, V, 4>
                                                                                                   : block_norm_kernel<T, V, kMaxPieces<T>>;
  else
    k = s.nv <= 2 ? block_norm_kernel<T, 1, 2> : s.nv <= 8 ? block_norm_kernel<T, 1, 8> : block_norm_kernel<T, 1, 32>;
  B200_CHECK_CUDA(launch_chained(k, dim3(grid), block, 0, st, p));
  return 0;
}

struct BwdShape {
  RowShape s;
  bool vec;
  int grid;
};
template <typename T>
BwdShape bwd_shape(const NormParams& p, bool vec) {
  constexpr int V = 16 / sizeof(T);
  BwdShape r;
  r.vec = vec;
  r.s = row_shape(vec ? p.H / V : p.H);
  r.grid = (int)std::min<int64_t>((p.T + r.s.rows - 1) / r.s.rows, device_sm_count());
  return r;
}

template <typename T>
int launch_norm_bwd_t(const NormBwdParams& b, const ColumnSumParams& sums, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const NormParams& p = b.f;
  const bool vec = vector_ok<T>(p) && aligned16(b.dh) && aligned16(b.dn) && aligned16(b.dy) && aligned16(b.dr) &&
                   (p.gate_kind == B200MOE_GATE_TOKEN || aligned16(b.dgate));
  BwdShape r = bwd_shape<T>(p, vec);
  const bool wide = 2 * ((p.H + 15) / 16) > kRowThreads && (p.H + 7) / 8 <= kWideThreads && ring_gate(p) == 0;
  const int values = wide ? 8 : 16, threads = wide ? kWideThreads : kRowThreads;
  const int arrays = 1 + (p.wn != nullptr && p.r != nullptr) + (b.dh != nullptr) + (b.dn != nullptr) + (p.gate_kind == B200MOE_GATE_FULL);
  const int row_bytes = arrays * p.H * (int)sizeof(T);
  const int tpr = (int)round_up64((p.H + values - 1) / values, 32);
  const bool ring = ring_ok<T>(p, vec) && tpr <= threads && 2 * row_bytes <= kRingLimit;
  void (*k)(NormBwdParams) = nullptr;
  if (ring) {
    const int per_sm = std::max(1, std::min(threads / tpr, kRingLimit / (2 * row_bytes + 2048)));
    r.grid = (int)std::min<int64_t>(p.T, (int64_t)device_sm_count() * per_sm);
    r.s.rows = 1;
    void (*kr)(NormBwdParams) = fp32_weights(p) ? bwd_ring<T, float>(p, wide) : bwd_ring<T, T>(p, wide);
    B200_CHECK_CUDA(cudaFuncSetAttribute(kr, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingLimit));
    B200_CHECK_CUDA(launch_chained(kr, dim3(r.grid), dim3(tpr), 2 * (size_t)row_bytes, st, b));
  } else if (vec)
    k = r.s.nv == 1 ? block_norm_bwd_kernel<T, V, 1> : r.s.nv == 2 ? block_norm_bwd_kernel<T, V, 2>
        : r.s.nv == 4 ? block_norm_bwd_kernel<T, V, 4> : block_norm_bwd_kernel<T, V, kMaxPieces<T>>;
  else
    k = r.s.nv <= 2 ? block_norm_bwd_kernel<T, 1, 2> : r.s.nv <= 8 ? block_norm_bwd_kernel<T, 1, 8> : block_norm_bwd_kernel<T, 1, 32>;
  if (!ring) B200_CHECK_CUDA(launch_chained(k, dim3(r.grid), dim3(r.s.tpr, r.s.rows), 0, st, b));
  if (b.part != nullptr) {
    ColumnSumParams c = sums;
    c.part = b.part;
    c.rows = r.grid * r.s.rows;
    c.H = p.H;
    B200_CHECK_CUDA(launch_chained(column_sum_kernel<T>, dim3((p.H + 31) / 32, 3), dim3(kSumGroups * 32), 0, st, c));
  }
  return 0;
}

}  // namespace

static int check_norm(int64_t y_stride, int64_t r_stride, int64_t gate_stride, int T, int H, int dtype, int gate_kind,
                      const void* gate) {
  B200_CHECK_ARG(T >= 0 && H >= 1 && H <= kMaxNormWidth, "block_norm: T=%d H=%d (H up to %d)", T, H, kMaxNormWidth);
  B200_CHECK_ARG(dtype >= B200MOE_T_BF16 && dtype <= B200MOE_T_FP32, "block_norm: dtype %d unknown", dtype);
  B200_CHECK_ARG(gate_kind >= B200MOE_GATE_NONE && gate_kind <= B200MOE_GATE_FULL, "block_norm: gate kind %d unknown", gate_kind);
  B200_CHECK_ARG(T == 0 || (gate_kind == B200MOE_GATE_NONE) == (gate == nullptr), "block_norm: gate and its kind disagree");
  B200_CHECK_ARG(y_stride >= 0 && r_stride >= 0 && gate_stride >= 0, "block_norm: negative row stride");
  return 0;
}

int64_t block_norm_bwd_workspace(int T, int H, int dtype) {
  // rows of partial sums: the largest of the shapes that a call of this size can take (the ring's CTAs hold 16 values a thread)
  const int ring_per_sm = std::max(1, kRowThreads / (int)round_up64((H + 15) / 16, 32));
  int64_t rows = std::min<int64_t>(T, (int64_t)device_sm_count() * ring_per_sm);
  for (int vec = 0; vec < 2; ++vec) {
    const RowShape s = row_shape(vec ? (H + (dtype == B200MOE_T_FP32 ? 3 : 7)) / (dtype == B200MOE_T_FP32 ? 4 : 8) : H);
    rows = std::max(rows, std::min<int64_t>((T + s.rows - 1) / s.rows, device_sm_count()) * s.rows);
  }
  return rows * 3 * H * (int64_t)sizeof(float);
}

}  // namespace b200moe

using namespace b200moe;

extern "C" {

int b200moe_block_norm(const void* y, int64_t y_stride, const void* residual, int64_t residual_stride, const void* weight,
                       const void* gate, int64_t gate_stride, const void* next_weight, int32_t T, int32_t H, int32_t dtype,
                       int32_t fp32_params, int32_t gate_kind, float residual_scale, float eps, void* h, void* n, void* q,
                       float* q_scale, float* rstd, void* stream) {
  if (int rc = check_norm(y_stride, residual_stride, gate_stride, T, H, dtype, gate_kind, gate)) return rc;
  B200_CHECK_ARG(n == nullptr || next_weight != nullptr, "block_norm: n needs next_weight");
  B200_CHECK_ARG((q == nullptr) == (q_scale == nullptr), "block_norm: q and q_scale go together");
  B200_CHECK_ARG(h != nullptr || n != nullptr || q != nullptr || T == 0, "block_norm: no output");
  if (T == 0) return 0;
  B200_CHECK_ARG(y != nullptr, "block_norm: NULL pointer");
  NormParams p = {y, residual, weight, gate, next_weight, y_stride, residual_stride, gate_stride, h, n, (int8_t*)q, q_scale, rstd,
                  T, H, gate_kind, fp32_params & 1, (fp32_params >> 1) & 1, (fp32_params >> 2) & 1, residual_scale, eps};
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == B200MOE_T_BF16 ? launch_norm_t<__nv_bfloat16>(p, st) : dtype == B200MOE_T_FP16 ? launch_norm_t<__half>(p, st)
                                                                                              : launch_norm_t<float>(p, st);
}

int b200moe_quantize_int8(const void* x, int64_t x_stride, int32_t T, int32_t K, int32_t dtype, void* q, float* scale,
                          void* stream) {
  B200_CHECK_ARG(T == 0 || (x && q && scale), "quantize_int8: NULL pointer");
  return b200moe_block_norm(x, x_stride, nullptr, 0, nullptr, nullptr, 0, nullptr, T, K, dtype, 0, B200MOE_GATE_NONE, 0.f, 0.f,
                            nullptr, nullptr, q, scale, nullptr, stream);
}

int b200moe_block_norm_bwd_workspace(int32_t T, int32_t H, int32_t dtype, int64_t* bytes) {
  B200_CHECK_ARG(bytes != nullptr && T >= 0 && H >= 1 && H <= kMaxNormWidth && dtype >= B200MOE_T_BF16 && dtype <= B200MOE_T_FP32,
                 "block_norm_bwd_workspace: T=%d H=%d dtype=%d", T, H, dtype);
  *bytes = block_norm_bwd_workspace(T, H, dtype);
  return 0;
}

int b200moe_block_norm_bwd(const void* y, int64_t y_stride, const void* residual, int64_t residual_stride, const void* weight,
                           const void* gate, int64_t gate_stride, const void* next_weight, int32_t T, int32_t H, int32_t dtype,
                           int32_t fp32_params, int32_t gate_kind, float residual_scale, const float* rstd, const void* dh,
                           const void* dn, void* dy, void* dresidual, void* dweight, void* dgate, void* dnext_weight,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_norm(y_stride, residual_stride, gate_stride, T, H, dtype, gate_kind, gate)) return rc;
  B200_CHECK_ARG((weight || !dweight) && (next_weight || !dnext_weight) && (gate || !dgate) && (residual || !dresidual),
                 "block_norm_bwd: the gradient of an absent tensor");
  B200_CHECK_ARG(dn == nullptr || next_weight != nullptr, "block_norm_bwd: dn needs next_weight");
  const bool channel = gate_kind == B200MOE_GATE_CHANNEL;
  const bool sums = dweight || dnext_weight || (channel && dgate);
  B200_CHECK_ARG(!sums || T == 0 || (workspace && workspace_bytes >= block_norm_bwd_workspace(T, H, dtype)),
                 "block_norm_bwd: workspace holds %lld bytes", (long long)workspace_bytes);
  cudaStream_t st = (cudaStream_t)stream;
  if (T == 0) {
    const size_t b = dtype == B200MOE_T_FP32 ? 4 : 2;
    if (dweight) B200_CHECK_CUDA(cudaMemsetAsync(dweight, 0, H * ((fp32_params & 1) ? 4 : b), st));
    if (channel && dgate) B200_CHECK_CUDA(cudaMemsetAsync(dgate, 0, H * ((fp32_params & 2) ? 4 : b), st));
    if (dnext_weight) B200_CHECK_CUDA(cudaMemsetAsync(dnext_weight, 0, H * ((fp32_params & 4) ? 4 : b), st));
    return 0;
  }
  B200_CHECK_ARG(y != nullptr && ((weight == nullptr && next_weight == nullptr) || rstd != nullptr), "block_norm_bwd: NULL pointer");
  NormBwdParams b;
  b.f = {y, residual, weight, gate, next_weight, y_stride, residual_stride, gate_stride, nullptr, nullptr, nullptr, nullptr,
         const_cast<float*>(rstd), T, H, gate_kind, fp32_params & 1, (fp32_params >> 1) & 1, (fp32_params >> 2) & 1, residual_scale, 0.f};
  b.dh = dh; b.dn = dn; b.dy = dy; b.dr = dresidual; b.dgate = channel ? nullptr : dgate;
  b.part = sums ? (float*)workspace : nullptr;
  b.want_dw = dweight != nullptr; b.want_dwn = dnext_weight != nullptr; b.want_dgc = channel && dgate != nullptr;
  ColumnSumParams c = {};
  c.dst[0] = dweight; c.dst[1] = dnext_weight; c.dst[2] = channel ? dgate : nullptr;
  c.f32[0] = fp32_params & 1; c.f32[1] = (fp32_params >> 2) & 1; c.f32[2] = (fp32_params >> 1) & 1;
  return dtype == B200MOE_T_BF16 ? launch_norm_bwd_t<__nv_bfloat16>(b, c, st)
         : dtype == B200MOE_T_FP16 ? launch_norm_bwd_t<__half>(b, c, st) : launch_norm_bwd_t<float>(b, c, st);
}

}  // extern "C"
