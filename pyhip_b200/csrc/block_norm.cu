// RMS norms after and before a block, with the branch's gate and the residual's scale, and the 8-bit token quantiser:
//   u = y * rstd(y) * w   (or y, without w)        rstd(v) = 1 / sqrt(mean(v^2) + eps)
//   h = alpha * r + g u                              g: none, or one value per channel, per token or per element
//   n = h * rstd(h) * w'                             stored in the rows' type or as 8-bit integers with the row's scale
// All of it in 32 bits from the inputs, rounded once where it is stored: n is the norm of the unrounded h.
//
// Bound by memory: forward reads y and r and writes h and n (8 bytes a value in 16-bit types), backward reads
// y, r, dh, dn and writes dy and dr (12 bytes).  A row stays in the registers of the threads that share it (each takes
// the same columns of every row, in 16-byte pieces), so every value is read and written once.
#include <algorithm>

#include "rowwise.cuh"

namespace b200moe {

namespace {

constexpr int kRowThreads = 512;          // threads of a CTA at most
constexpr int kMaxNormWidth = 16384;
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

// Backward.  With e = dh + rstd(h) w' dn and c = rstd(h)^3 mean(w' dn h) the gradient that reaches h is e - c h, and the
// sum that the norm of y needs, sum(w y g (e - c h)), is A - c B with A = sum(w y g e), B = sum(w y g h): all three sums
// of a row are formed in one reduction.  A gate per token is a factor of A and B, and its own gradient is rstd(y)(A - cB).
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
          const float wy = y[i][j] * w[j];
          h[i][j] = fmaf(p.alpha, h[i][j], g[j] * (wy * ry));
          const float wd = wn[j] * dn[i][j];
          e[i][j] = fmaf(rh, wd, e[i][j]);
          s[0] = fmaf(wd, h[i][j], s[0]);
          const float v = by_value ? wy * g[j] : wy;
          s[1] = fmaf(v, e[i][j], s[1]);
          s[2] = fmaf(v, h[i][j], s[2]);
        }
      }
    }
    red.sum(s);
    const float c3 = rh * rh * rh * s[0] * inv_h;
    const float raw = s[1] - c3 * s[2];
    const float cy = (p.w != nullptr) ? ry * ry * ry * (by_value ? raw : gt * raw) * inv_h : 0.f;
    if (row && threadIdx.x == 0 && p.gate_kind == B200MOE_GATE_TOKEN && b.dgate != nullptr) {
      const float one[1] = {ry * raw};
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
          const float d = fmaf(-c3, h[i][j], e[i][j]);
          dr[j] = p.alpha * d;
          const float du = d * g[j], yr = y[i][j] * ry;
          out[j] = fmaf(ry * w[j], du, -cy * y[i][j]);
          aw[i][j] = fmaf(du, yr, aw[i][j]);
          an[i][j] = fmaf(dn[i][j], h[i][j] * rh, an[i][j]);
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

// dst[c] = sum over the partial rows, in ascending order within eight interleaved groups that are then added in order.
struct ColumnSumParams {
  const float* part;
  void* dst[3];
  int f32[3];
  int rows, H;
};
template <typename T>
__global__ void __launch_bounds__(256)
column_sum_kernel(const __grid_constant__ ColumnSumParams p) {
  __shared__ float s[8][33];
  grid_dep_wait();
  grid_dep_launch();
  const int which = blockIdx.y, col = blockIdx.x * 32 + (threadIdx.x & 31), grp = threadIdx.x >> 5;
  if (p.dst[which] == nullptr) return;
  float a = 0.f;
  if (col < p.H)
    for (int r = grp; r < p.rows; r += 8) a += p.part[((int64_t)r * 3 + which) * p.H + col];
  s[grp][threadIdx.x & 31] = a;
  __syncthreads();
  if (grp == 0 && col < p.H) {
    float v[1] = {0.f};
#pragma unroll
    for (int g = 0; g < 8; ++g) v[0] += s[g][threadIdx.x];
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

template <typename T>
int launch_norm_t(const NormParams& p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = vector_ok<T>(p);
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
  const BwdShape r = bwd_shape<T>(p, vec);
  void (*k)(NormBwdParams) = nullptr;
  if (vec)
    k = r.s.nv == 1 ? block_norm_bwd_kernel<T, V, 1> : r.s.nv == 2 ? block_norm_bwd_kernel<T, V, 2>
        : r.s.nv == 4 ? block_norm_bwd_kernel<T, V, 4> : block_norm_bwd_kernel<T, V, kMaxPieces<T>>;
  else
    k = r.s.nv <= 2 ? block_norm_bwd_kernel<T, 1, 2> : r.s.nv <= 8 ? block_norm_bwd_kernel<T, 1, 8> : block_norm_bwd_kernel<T, 1, 32>;
  B200_CHECK_CUDA(launch_chained(k, dim3(r.grid), dim3(r.s.tpr, r.s.rows), 0, st, b));
  if (b.part != nullptr) {
    ColumnSumParams c = sums;
    c.part = b.part;
    c.rows = r.grid * r.s.rows;
    c.H = p.H;
    B200_CHECK_CUDA(launch_chained(column_sum_kernel<T>, dim3((p.H + 31) / 32, 3), dim3(256), 0, st, c));
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
  // rows of partial sums: the larger of the two shapes that a call of this size can take
  int64_t rows = 0;
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
