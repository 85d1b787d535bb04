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

// 16 bytes, global to shared, asynchronously; groups complete in order, and a thread that reads only what it copied itself
// needs no barrier
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}

// Two fp32 values to an instruction (fma.rn.f32x2): the row kernels are close to the issue rate, not to the FMA rate.  A pair
// is one 64-bit value, so that it stays in a pair of neighbouring registers.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 split(f32x2 v) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
  return d;
}
__device__ __forceinline__ float both_of(f32x2 v) {
  const float2 d = split(v);
  return d.x + d.y;
}
__device__ __forceinline__ f32x2 both(float v) { return pair(v, v); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// 16 bytes of a row's type <-> pairs of fp32
template <typename T> constexpr int kPairs = 8 / (int)sizeof(T);
__device__ __forceinline__ void unpack16(const uint4& v, f32x2 (&o)[2], float) {
  o[0] = pair(__uint_as_float(v.x), __uint_as_float(v.y));
  o[1] = pair(__uint_as_float(v.z), __uint_as_float(v.w));
}
__device__ __forceinline__ void unpack16(const uint4& v, f32x2 (&o)[4], __nv_bfloat16) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ void unpack16(const uint4& v, f32x2 (&o)[4], __half) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    o[i] = pair(f.x, f.y);
  }
}
__device__ __forceinline__ uint4 pack16(const f32x2 (&v)[2], float) {
  const float2 a = split(v[0]), b = split(v[1]);
  return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
}
__device__ __forceinline__ uint4 pack16(const f32x2 (&v)[4], __nv_bfloat16) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 k = __float22bfloat162_rn(split(v[i]));
    w[i] = *reinterpret_cast<const uint32_t*>(&k);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack16(const f32x2 (&v)[4], __half) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 k = __float22half2_rn(split(v[i]));
    w[i] = *reinterpret_cast<const uint32_t*>(&k);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// the parameters of piece c of a row of T, held as T or as fp32
template <typename T, typename P, int N2>
__device__ __forceinline__ void load_piece(const void* p, int c, f32x2 (&o)[N2]) {
  static_assert(N2 == kPairs<T>, "a piece of the row's type");
  if constexpr (sizeof(P) == sizeof(T)) {
    unpack16(static_cast<const uint4*>(p)[c], o, T());
  } else {
    const float4 a = static_cast<const float4*>(p)[2 * c], b = static_cast<const float4*>(p)[2 * c + 1];
    o[0] = pair(a.x, a.y); o[1] = pair(a.z, a.w);
    o[2] = pair(b.x, b.y); o[3] = pair(b.z, b.w);
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

// Sums of four values over a warp with six exchanges: two lanes swap what the other keeps, so the values thin out while
// the lanes are joined.  Lane l ends with the sum of value l & 3.
__device__ __forceinline__ float warp_sum4(float a, float b, float c, float d) {
  const int lane = threadIdx.x & 31;
  const bool o1 = lane & 1, o2 = lane & 2;
  float x = o1 ? b : a, y = o1 ? d : c;
  x += __shfl_xor_sync(0xffffffffu, o1 ? a : b, 1);
  y += __shfl_xor_sync(0xffffffffu, o1 ? c : d, 1);
  float v = o2 ? y : x;
  v += __shfl_xor_sync(0xffffffffu, o2 ? x : y, 2);
#pragma unroll
  for (int k = 4; k < 32; k <<= 1) v += __shfl_xor_sync(0xffffffffu, v, k);
  return v;
}

// The same for CTAs whose threads all share the row.
struct CtaReduce {
  float* slots;   // [2][32][4], 16-byte aligned; the entries of warps that do not exist stay zero
  uint32_t turn;
  __device__ explicit CtaReduce(float* s) : slots(s), turn(0) {
    for (int i = threadIdx.x; i < 2 * 32 * 4; i += blockDim.x) s[i] = 0.f;
    __syncthreads();
  }
  __device__ __forceinline__ float sum(float v) {
    v = warp_sum(v);
    float* s = slots + turn * 128;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    // the warps' sums, four at a time
    const float4* q = reinterpret_cast<const float4*>(s);
    float4 a = q[0];
    for (int k = 1; k < ((int)blockDim.x + 127) / 128; ++k) {
      const float4 b = q[k];
      a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
    }
    return (a.x + a.y) + (a.z + a.w);
  }
  // (the slots of a turn belong to one kind of reduction in a kernel: sum3 here, sum and max_u32 elsewhere)
  __device__ __forceinline__ void sum3(float& a, float& b, float& c) {
    const int lane = threadIdx.x & 31;
    float v = warp_sum4(a, b, c, 0.f);
    float* s = slots + turn * 128;
    turn ^= 1;
    if (lane < 4) s[(threadIdx.x >> 5) * 4 + lane] = v;
    __syncthreads();
    const float4 q = reinterpret_cast<const float4*>(s)[lane];
    v = warp_sum4(q.x, q.y, q.z, q.w);
    a = __shfl_sync(0xffffffffu, v, 0);
    b = __shfl_sync(0xffffffffu, v, 1);
    c = __shfl_sync(0xffffffffu, v, 2);
  }
  __device__ __forceinline__ uint32_t max_u32(uint32_t v) {
    uint32_t* s = reinterpret_cast<uint32_t*>(slots + turn * 128);
    turn ^= 1;
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    const uint4* q = reinterpret_cast<const uint4*>(s);
    v = 0;
    for (int k = 0; k < ((int)blockDim.x + 127) / 128; ++k) {
      const uint4 b = q[k];
      v = max(v, max(max(b.x, b.y), max(b.z, b.w)));
    }
    return v;
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

// max(|a|, |b|) in magnitude (the sign means nothing), NaN if either is
__device__ __forceinline__ float max_abs_nan(float a, float b) {
  float d;
  asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
template <int N2>
__device__ __forceinline__ float max_abs_nan(float m, const f32x2 (&v)[N2]) {
#pragma unroll
  for (int j = 0; j < N2; ++j) {
    const float2 x = split(v[j]);
    m = max_abs_nan(max_abs_nan(m, x.x), x.y);
  }
  return m;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// 2 N2 values to 8-bit integers, four to a word.  v * inv + 1.5 * 2^23 holds the nearest whole number in its low bits (the
// conversions between float and integer run at an eighth of the rate); where a remainder reaches s/2 the exact rule above
// decides again, which is rare.
template <int N2>
__device__ __forceinline__ void quant_int8(const f32x2 (&v)[N2], float s, float inv, uint32_t (&out)[N2 / 2]) {
  const f32x2 inv2 = both(inv), magic = both(12582912.f), minus = both(-12582912.f), ms = both(-s);
  uint32_t b[2 * N2];
  float worst = 0.f;
#pragma unroll
  for (int j = 0; j < N2; ++j) {
    const f32x2 m = fma2(v[j], inv2, magic);
    const float2 k = split(m), d = split(fma2(add2(m, minus), ms, v[j]));
    b[2 * j] = __float_as_uint(k.x);
    b[2 * j + 1] = __float_as_uint(k.y);
    worst = fmaxf(fmaxf(worst, fabsf(d.x)), fabsf(d.y));
  }
  if (worst >= 0.5f * s) {
#pragma unroll
    for (int j = 0; j < N2; ++j) {
      const float2 x = split(v[j]);
      b[2 * j] = (uint32_t)quant_int8(x.x, s, inv);
      b[2 * j + 1] = (uint32_t)quant_int8(x.y, s, inv);
    }
  }
#pragma unroll
  for (int j = 0; j < N2 / 2; ++j)
    out[j] = __byte_perm(__byte_perm(b[4 * j], b[4 * j + 1], 0x0040), __byte_perm(b[4 * j + 2], b[4 * j + 3], 0x0040), 0x5410);
}

}  // namespace b200moe
