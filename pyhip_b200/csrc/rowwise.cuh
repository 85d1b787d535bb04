// Helpers of the row-wise kernels (norms, 8-bit quantiser, router): vector access to rows of bf16, fp16 or fp32 with
// 32-bit arithmetic, row sums over the threads that share a row, and the rounding to 8-bit integers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "ptx_sm100.cuh"

namespace b200moe {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ void load_f(const T* p, float (&o)[N]) {
  const Pack<T, N> k = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = to_f(k.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_f(T* p, const float (&v)[N]) {
  Pack<T, N> k;
#pragma unroll
  for (int i = 0; i < N; ++i) k.v[i] = from_f<T>(v[i]);
  *reinterpret_cast<Pack<T, N>*>(p) = k;
}
// N values of a parameter that is held in the rows' type or in fp32 (16 bytes at a time at most)
template <typename T, int N>
__device__ __forceinline__ void load_param(const void* p, bool f32, int64_t at, float (&o)[N]) {
  if (f32) {
    constexpr int M = N < 4 ? N : 4;
#pragma unroll
    for (int i = 0; i < N; i += M) {
      float q[M];
      load_f<float, M>(static_cast<const float*>(p) + at + i, q);
#pragma unroll
      for (int j = 0; j < M; ++j) o[i + j] = q[j];
    }
  } else {
    load_f<T, N>(static_cast<const T*>(p) + at, o);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_param(void* p, bool f32, int64_t at, const float (&v)[N]) {
  if (f32) {
    constexpr int M = N < 4 ? N : 4;
#pragma unroll
    for (int i = 0; i < N; i += M) {
      float q[M];
#pragma unroll
      for (int j = 0; j < M; ++j) q[j] = v[i + j];
      store_f<float, M>(static_cast<float*>(p) + at + i, q);
    }
  } else {
    store_f<T, N>(static_cast<T*>(p) + at, v);
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Sums (or the unsigned maximum) over the threads that share a row: blockDim.x threads, a whole number of warps, of
// the blockDim.y rows of a CTA.  Two slots used in turn make one barrier enough: a slot is written again only after
// the barrier of the reduction in between, which every reader of the slot has passed.
constexpr int kMaxRowWarps = 32;   // warps of a CTA
struct RowReduce {
  float* slots;   // [2][3][kMaxRowWarps]
  uint32_t turn;
  __device__ explicit RowReduce(float* s) : slots(s), turn(0) {}
  template <int N>
  __device__ __forceinline__ void sum(float (&v)[N]) {
    static_assert(N <= 3, "three sums at most");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    const int wpr = blockDim.x >> 5;
    if (wpr == 1) return;
    float* s = slots + turn * 3 * kMaxRowWarps;
    turn ^= 1;
    const int w0 = threadIdx.y * wpr;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[i * kMaxRowWarps + w0 + (threadIdx.x >> 5)] = v[i];
    }
    __syncthreads();
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < wpr ? s[i * kMaxRowWarps + w0 + lane] : 0.f);
  }
  __device__ __forceinline__ uint32_t max_u32(uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    const int wpr = blockDim.x >> 5;
    if (wpr == 1) return v;
    uint32_t* s = reinterpret_cast<uint32_t*>(slots + turn * 3 * kMaxRowWarps);
    turn ^= 1;
    const int w0 = threadIdx.y * wpr;
    if ((threadIdx.x & 31) == 0) s[w0 + (threadIdx.x >> 5)] = v;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    return __reduce_max_sync(0xffffffffu, lane < wpr ? s[w0 + lane] : 0u);
  }
};

// Scale of a row of 8-bit integers from the largest magnitude's bits: max(fl32(amax / 127), 2^-100); NaN where the row
// holds an infinity or NaN (the unsigned maximum of the magnitudes' bits keeps both), so that its products are NaN too.
__device__ __forceinline__ float int8_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return fmaxf(__fdiv_rn(__uint_as_float(amax_bits), 127.f), 7.888609052210118e-31f);
}
// The whole number nearest to v / s, ties to even, exactly: v * (1/s) is off by two roundings and may land on the
// wrong side of a border, so the remainder v - q s decides.  It is exact in 32 bits (v and s are multiples of 2^-24 s
// where |v| >= s/2, and it is at most about s/2), hence so is its comparison with s/2.
__device__ __forceinline__ int quant_int8(float v, float s, float inv) {
  float q = rintf(v * inv);
  const float d = fmaf(-q, s, v), half = 0.5f * s, ad = fabsf(d);
  const int qi = (int)q;
  const bool off = ad > half || (ad == half && (qi & 1));
  return off ? qi + (d > 0.f ? 1 : -1) : qi;
}

}  // namespace b200moe
