// W8A8 linear layer: y[t, n] = (sum_k q[t, k] W[n, k]) * s_t * w_n (+ b_n), 8-bit integers with one fp32 scale per token
// and per output channel.  tcgen05.mma kind::i8, int32 accumulators in tensor memory: the sum is exact (K < 2^17), so
// splitting K over CTAs changes no bit of the result.
//
// Two kernels, chosen by size (pick_variant):
//   split   one 128-feature x BT-token tile per CTA, the weights on the MMA's M side; the CTAs of a cluster take equal
//           ranges of K and add their tiles through distributed shared memory.  For few tokens, where the weights' bytes
//           and the launch latency bound the call: every weight byte is requested as soon as the CTA starts.  A single
//           token is quantised here too, by the epilogue warps while the weights are on their way: every CTA reads the row
//           for its scale and converts its own range of K (one launch instead of two and no workspace, the same time on
//           the GPU, 3.3 us less on the host; from two tokens on the repeated reading costs the GPU more).
//   pair    persistent CTA pairs (cta_group::2), 256 tokens x BN features a tile: each CTA holds its 128 tokens' rows and
//           half of the feature rows, two accumulators overlap a tile's epilogue with the next one's products.
//
// On a B200 (tokens, weight N x K): 1, 2880 x 2880 6.2-6.6 us; 64, 14336 x 4096 15.4 us (17.3 with the quantiser; the weights'
// stream alone is 9); 64, 4096 x 4096 10 us; 512, 4096 x 4096 12.9 us; 1000, 2048 x 7168 17.6 us; 2048, 7168 x 4096 43 us;
// 16384, 14336 x 4096 575-606 us, 3.2-3.3 POP/s (tensor pipe 89 % active at 2048 tokens, 2.95 POP/s).  What a call does not overlap, 6 to 7 us, bounds the small
// ones: start and first load 2, the last tile's way out and the join 3 to 4.
//
// A pipeline stage is 128 bytes of K (one swizzle span): 128 rows of one operand and BT or BN/2 rows of the other, one TMA
// copy each; K and row tails are zero-filled by the copy.  Every barrier wait is bounded; one that runs out sets status[],
// what its sums belong to becomes NaN, and the CTA unwinds and frees its tensor memory.
#include <string.h>

#include <algorithm>

#include "gemm_common.cuh"
#include "rowwise.cuh"

namespace b200moe {

namespace {

constexpr int kThreadsI8 = 192;                 // warp 0 TMA producer, warp 1 MMA issuer, warps 2-5 epilogue
constexpr int kTileKI8 = 128;                   // bytes of K per stage
constexpr int kRowTile = 128;                   // rows of the M-side operand per CTA
constexpr int kRowTileBytes = kRowTile * kTileKI8;
constexpr int kMaxStagesI8 = 12;
constexpr int kMaxTokenTile = 128;              // split: a lane holds a token column's scale for every 32 of them
constexpr int kSmemLimitI8 = 232448;            // 227 KB
constexpr int kCtlBytes = 1024;
constexpr int kPairThreads = 320;               // the same with eight epilogue warps, 2-9
constexpr int kStoreCols = 32;                  // columns of a staged store: 64 bytes of a 16-bit type
constexpr int kStagingBytes = 32 * 64;          // 32 rows of them
constexpr int kPairScaleBytes = 2 * 2 * 256 * 4;   // two tiles' channel scales and biases

struct LinearParams {
  CUtensorMap tmX;      // token rows (K, T)
  CUtensorMap tmW;      // weight rows (K, N)
  CUtensorMap tmY;      // output (N, T), box 32 x 32; only when store_tma
  const float* x_scale;
  const float* w_scale;
  const float* bias;
  void* y;
  int32_t* status;
  const void* x;        // the row that the split kernel quantises itself
  int T, N, K, KB, k_tail_steps, stages, fp16, store_tma, early_weights, x_dtype, x_vec;
  int hold_back;                  // the CTAs (along x) that leave out their last weight copy (-1: none), for tests of the waits
  int tokens, splits;             // split: token tile, CTAs that share K
  int m_tiles, n_tiles;           // pair
};

// Where a bounded wait that ran out is reported if the caller gives no words of its own: one pair per device, zero when the library
// is loaded, there for calls that are captured too, and never cleared.
__device__ int32_t g_linear_status[2];
__device__ __forceinline__ void report_abort(const LinearParams& p, uint32_t word) {
  int32_t* s = p.status != nullptr ? p.status : g_linear_status;
  s[0] = (int32_t)word;
  s[1] = (int32_t)blockIdx.x;
}

struct SmemCtlI8 {
  uint64_t full[kMaxStagesI8];
  uint64_t empty[kMaxStagesI8];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint32_t tmem_base;
  uint32_t abort_word;
  uint32_t peer_lost;             // a CTA of the cluster has no sums to give
};
static_assert(sizeof(SmemCtlI8) <= kCtlBytes, "control block");

// Instruction descriptor of kind::i8: [4,6) D format (2 = s32)  [7,10) A format  [10,13) B format (1 = signed 8-bit)
// [17,23) N>>3  [24,29) M>>4; both operands K-major
__device__ __forceinline__ uint32_t make_idesc_i8(uint32_t M, uint32_t N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
// D[tmem] (+)= A[smem] * B[smem]^T, signed 8-bit x signed 8-bit, K = 32 per instruction
template <bool PAIR>
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], da, db, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw)
        : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
// into this CTA's shared memory, completing bytes on the pair's leading CTA's barrier
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar & kLeaderMask), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src), "r"(c0),
               "r"(c1)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer_smem(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ int4 ld_peer_v4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t ld_peer_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_peer_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_peer_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint32_t pack2(float a, float b, bool fp16) {
  if (fp16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// let this CTA's copies still in flight land before shared memory is released (bounded)
__device__ __forceinline__ void drain_copies(SmemCtlI8* ctl, int64_t issued, int S) {
  for (int64_t i = issued > S ? issued - S : 0; i < issued; ++i) {
    const uint32_t bar = smem_u32(&ctl->full[i % S]);
    const uint64_t t0 = global_timer_ns();
    while (!mbar_try_wait(bar, (uint32_t)((i / S) & 1)) && global_timer_ns() - t0 < 200000000ull) {}
  }
}

// ------------------------------------------------------------------------------------ split
constexpr int kFusedTile = 16;                  // token tile of the MMA where the split kernel quantises its one row itself
constexpr int kFusedBlockBytes = kFusedTile * kTileKI8;
constexpr int kFusedBlocks = 16;                // k-blocks of a CTA, at most
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// 16 neighbouring values of a row as pairs
template <typename T>
__device__ __forceinline__ void load_16(const T* src, bool vec, f32x2 (&v)[8]) {
  if (vec) {
    constexpr int P = kPairs<T>;
#pragma unroll
    for (int i = 0; i < 8 / P; ++i) {
      f32x2 part[P];
      unpack16(reinterpret_cast<const uint4*>(src)[i], part, T());
#pragma unroll
      for (int j = 0; j < P; ++j) v[i * P + j] = part[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = pair(to_f(src[2 * i]), to_f(src[2 * i + 1]));
  }
}
// The epilogue warps' part of the fused split kernel: the row's scale, then this CTA's k-blocks of the row as the MMA's N-side
// tiles (16 rows of 128 bytes in the 128-byte swizzle, all but the first of them zero).
template <typename T>
__device__ __forceinline__ void quantise_row(const LinearParams& p, uint32_t tiles, int kb0, int blocks, uint32_t* maxima, float* scale) {
  const int te = (int)threadIdx.x - 64;
  const T* x = static_cast<const T*>(p.x);
  const bool vec = p.x_vec != 0;
  float m = 0.f;
#pragma unroll 4
  for (int c = te; c < p.K / 16; c += 128) {
    f32x2 v[8];
    load_16<T>(x + c * 16, vec, v);
    m = max_abs_nan(m, v);
  }
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(m) & 0x7fffffffu);
  if ((te & 31) == 0) maxima[te >> 5] = bits;
  for (int i = te; i < blocks * (kFusedBlockBytes / 16); i += 128)
    if ((i & 127) >= 8) st_shared_v4(tiles + (uint32_t)i * 16, 0, 0, 0, 0);          // rows 1 to 15 of each tile
  epilogue_sync();
  const float s = int8_scale(max(max(maxima[0], maxima[1]), max(maxima[2], maxima[3])));
  if (te == 0) *scale = s;
  for (int c = te; c < blocks * 8; c += 128) {             // 16-byte pieces of the row in this CTA's range
    const int k = kb0 * kTileKI8 + c * 16;
    uint32_t o[4] = {0, 0, 0, 0};
    if (k < p.K && s == s) {                               // (a row with an infinity or NaN: zeros, and scale NaN)
      f32x2 v[8];
      load_16<T>(x + k, vec, v);
      quant_int8(v, s, __fdividef(1.f, s), o);
    }
    st_shared_v4(tiles + (uint32_t)(c >> 3) * kFusedBlockBytes + (uint32_t)((c & 7) << 4), o[0], o[1], o[2], o[3]);
  }
}

template <bool FUSED>
__global__ void __launch_bounds__(kThreadsI8)
linear_int8_split_kernel(const __grid_constant__ LinearParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint32_t maxima[4];
  __shared__ float row_scale;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  SmemCtlI8* ctl = reinterpret_cast<SmemCtlI8*>(smem);
  const uint32_t stage0 = smem_u32(smem) + kCtlBytes;
  const int S = p.stages, BT = p.tokens, C = p.splits;
  const uint32_t stage_bytes = (uint32_t)(kRowTileBytes + (FUSED ? 0 : BT * kTileKI8));
  const uint32_t token_tiles = stage0 + S * stage_bytes;   // FUSED: one for each k-block of the CTA
  const uint32_t cols = (uint32_t)max(32, BT);             // BT is 16, 32, 64 or 128
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)(blockIdx.x % (unsigned)C);        // clusters run along x
  const int n0 = (int)(blockIdx.x / (unsigned)C) * kRowTile, t0 = (int)blockIdx.y * BT;
  const int kb0 = (int)((int64_t)p.KB * rank / C), kb1 = (int)((int64_t)p.KB * (rank + 1) / C);
  volatile uint32_t* abort_word = &ctl->abort_word;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(smem_u32(&ctl->full[s]), 1);
      mbar_init(smem_u32(&ctl->empty[s]), 1);
    }
    mbar_init(smem_u32(&ctl->tmem_full[0]), 1);
    mbar_init(smem_u32(&ctl->tmem_empty[0]), 1);           // FUSED: the token tiles are ready
    ctl->abort_word = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&ctl->tmem_base), cols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = ctl->tmem_base;

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      // The weights do not depend on the launch in front when that is this call's own quantiser (early_weights): it
      // lets this grid start only after everything before it has completed.
      int ahead = 0;
      const int held = p.hold_back == (int)blockIdx.x ? kb1 - 1 : kb1;             // the k-block that is not fetched
      if (!FUSED && p.early_weights)
        for (; ahead < min(S, kb1 - kb0); ++ahead) {
          const uint32_t full = smem_u32(&ctl->full[ahead]);
          mbar_expect_tx(full, stage_bytes);
          if (kb0 + ahead < held) tma_load_2d(stage0 + ahead * stage_bytes, &p.tmW, full, (kb0 + ahead) * kTileKI8, n0);
        }
      grid_dep_wait();
      int64_t issued = 0;
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(smem_u32(&ctl->empty[stage]), phase ^ 1, abort_word, 0x1100 + stage)) { ok = false; break; }
        const uint32_t st = stage0 + stage * stage_bytes, full = smem_u32(&ctl->full[stage]);
        if (kb - kb0 >= ahead) {
          mbar_expect_tx(full, stage_bytes);
          if (kb < held) tma_load_2d(st, &p.tmW, full, kb * kTileKI8, n0);
        }
        if (!FUSED) tma_load_2d(st + kRowTileBytes, &p.tmX, full, kb * kTileKI8, t0);
        ++issued;
        if (++stage == S) { stage = 0; phase ^= 1; }
      }
      if (!ok || *abort_word) drain_copies(ctl, issued, S);
    }
  } else if (warp == 1) {
    const uint32_t idesc = make_idesc_i8(kRowTile, (uint32_t)BT);
    int stage = 0;
    uint32_t phase = 0;
    if (FUSED) ok = mbar_wait(smem_u32(&ctl->tmem_empty[0]), 0, abort_word, 0x1400);
    for (int kb = kb0; kb < kb1 && ok; ++kb) {
      if (!mbar_wait(smem_u32(&ctl->full[stage]), phase, abort_word, 0x1200 + stage)) { ok = false; break; }
      tc_fence_after_sync();
      __syncwarp();
      if (elect_one()) {
        const uint32_t st = stage0 + stage * stage_bytes;
        const uint32_t a_lo = desc_lo_sw(st), b_lo = desc_lo_sw(FUSED ? token_tiles + (uint32_t)(kb - kb0) * kFusedBlockBytes : st + kRowTileBytes);
        const int steps = kb == p.KB - 1 ? p.k_tail_steps : 4;
#pragma unroll
        for (int s = 0; s < 4; ++s)
          if (s < steps) umma_i8<false>(tmem_base, a_lo + 2 * s, b_lo + 2 * s, idesc, (kb != kb0 || s != 0) ? 1u : 0u);
        tc_commit(smem_u32(&ctl->empty[stage]));
        if (kb == kb1 - 1) tc_commit(smem_u32(&ctl->tmem_full[0]));
      }
      __syncwarp();
      if (++stage == S) { stage = 0; phase ^= 1; }
    }
    grid_dep_wait();
  } else {
    grid_dep_wait();
    if (FUSED) {
      if (p.x_dtype == B200MOE_T_BF16) quantise_row<__nv_bfloat16>(p, token_tiles, kb0, kb1 - kb0, maxima, &row_scale);
      else if (p.x_dtype == B200MOE_T_FP16) quantise_row<__half>(p, token_tiles, kb0, kb1 - kb0, maxima, &row_scale);
      else quantise_row<float>(p, token_tiles, kb0, kb1 - kb0, maxima, &row_scale);
      fence_proxy_async_smem();
      epilogue_sync();
      if (threadIdx.x == 64) mbar_arrive(smem_u32(&ctl->tmem_empty[0]));
    }
  }
  grid_dep_launch();

  // what the sums are multiplied by, on its way while the products are finished: a lane's four features, and the token
  // columns' scales spread over the lanes (the producer's other lanes have not waited for the launch in front yet)
  grid_dep_wait();
  const int live = min(BT, p.T - t0);
  const int n = n0 + lane * 4;
  float ws[4], bs[4], xs_of[kMaxTokenTile / 32];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ws[j] = n + j < p.N ? p.w_scale[n + j] : 0.f;
    bs[j] = (p.bias != nullptr && n + j < p.N) ? p.bias[n + j] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < kMaxTokenTile / 32; ++j) xs_of[j] = (!FUSED && j * 32 + lane < live) ? p.x_scale[t0 + j * 32 + lane] : 0.f;
  // the tile as [token][feature] int32 in the stages' memory, which the products no longer need
  if (warp >= 2) {
    ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&ctl->tmem_full[0]), 0, abort_word, 0x1300));
    if (ok) {
      tc_fence_after_sync();
      const int quad = warp & 3;
      const uint32_t at = stage0 + (uint32_t)(quad * 32 + lane) * 4;
      for (int c0 = 0; c0 < live; c0 += 16) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(tmem_base + ((uint32_t)(quad * 32) << 16) + c0, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) st_shared_u32(at + (uint32_t)(c0 + i) * (kRowTile * 4), v[i]);
      }
    }
  }
  // Tensor memory goes back before the CTA waits for the others of its cluster: an allocation blocks until there are columns, so a
  // CTA that kept its own here could wait for one that never gets any.  Warp 1 has nothing to hand over and frees them meanwhile.
  __syncwarp();
  tc_fence_before_sync();
  if (warp >= 2) asm volatile("bar.arrive 2, 160;" ::: "memory");
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  if (warp == 1) {
    asm volatile("bar.sync 2, 160;" ::: "memory");
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, cols);
    __syncwarp();
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  // token columns are dealt out over the cluster's warps; a lane adds four neighbouring features of all its CTAs.  Four
  // columns at a time: a load from another CTA takes hundreds of cycles.
  // A CTA whose wait ran out has no sums to give: the cluster's tile becomes NaN, as a row that cannot be quantised does.
  const bool lost = __any_sync(0xffffffffu, lane < C && ld_peer_u32(peer_smem(smem_u32(&ctl->abort_word), (uint32_t)min(lane, C - 1))) != 0);
  const int stride = C * (kThreadsI8 / 32);
  for (int c0 = rank + C * warp; c0 < live; c0 += 4 * stride) {
    int4 a[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) a[q] = make_int4(0, 0, 0, 0);
    for (int r = 0; r < C; ++r) {
      const uint32_t at = peer_smem(stage0 + (uint32_t)c0 * (kRowTile * 4) + lane * 16, (uint32_t)r);
      int4 v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = c0 + q * stride < live ? ld_peer_v4(at + (uint32_t)(q * stride) * (kRowTile * 4)) : make_int4(0, 0, 0, 0);
#pragma unroll
      for (int q = 0; q < 4; ++q) { a[q].x += v[q].x; a[q].y += v[q].y; a[q].z += v[q].z; a[q].w += v[q].w; }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = c0 + q * stride;
      if (c >= live) break;                                  // (the same for the whole warp)
      float xs = FUSED ? row_scale : __shfl_sync(0xffffffffu, c < 32 ? xs_of[0] : c < 64 ? xs_of[1] : c < 96 ? xs_of[2] : xs_of[3], c & 31);
      if (lost) xs = __uint_as_float(0x7fc00000u);
      const float o0 = fmaf((float)a[q].x * xs, ws[0], bs[0]), o1 = fmaf((float)a[q].y * xs, ws[1], bs[1]);
      const float o2 = fmaf((float)a[q].z * xs, ws[2], bs[2]), o3 = fmaf((float)a[q].w * xs, ws[3], bs[3]);
      const uint32_t lo = pack2(o0, o1, p.fp16), hi = pack2(o2, o3, p.fp16);
      uint16_t* dst = static_cast<uint16_t*>(p.y) + (int64_t)(t0 + c) * p.N + n;
      if ((p.N & 3) == 0) {
        if (n < p.N) *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
      } else {
        if (n < p.N) dst[0] = (uint16_t)lo;
        if (n + 1 < p.N) dst[1] = (uint16_t)(lo >> 16);
        if (n + 2 < p.N) dst[2] = (uint16_t)hi;
        if (n + 3 < p.N) dst[3] = (uint16_t)(hi >> 16);
      }
    }
  }
  if (threadIdx.x == 0 && ctl->abort_word != 0) report_abort(p, ctl->abort_word);
  __syncwarp();
  cluster_sync_all();                // no CTA leaves while another one reads its tile
}

// ------------------------------------------------------------------------------------ pair
// tile order: bands of eight token tiles, features running slowest inside a band, so that the CTAs at work at a time share
// both operands' rows in L2
__device__ __forceinline__ void tile_of(int w, int m_tiles, int n_tiles, int& m, int& n) {
  constexpr int BAND = 8;
  const int band = w / (BAND * n_tiles), first = band * BAND;
  const int height = min(BAND, m_tiles - first);
  const int in = w - first * n_tiles;
  m = first + in % height;
  n = in / height;
}

// arrive on the barrier at this offset in both CTAs of pair `z` of the cluster once the products issued so far are done
__device__ __forceinline__ void commit_to_pair(uint32_t bar, uint32_t z) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"((unsigned short)(3u << (2 * z)))
               : "memory");
}

// Z pairs of a cluster share one tile's K (Z = 1: persistent, a cluster walks over tiles).  With Z > 1 each pair ends up with
// BN / Z columns of the tile: the others' partial sums of them arrive in its stages' memory, one slot for each.
template <int BN, int Z>
__global__ void __launch_bounds__(kPairThreads, 1)
linear_int8_pair_kernel(const __grid_constant__ LinearParams p) {
  constexpr uint32_t B_BYTES = BN / 2 * kTileKI8, STAGE = kRowTileBytes + B_BYTES;
  constexpr uint32_t COLS = (Z == 1 ? 2 : 1) * BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  SmemCtlI8* ctl = reinterpret_cast<SmemCtlI8*>(smem);
  const int S = p.stages;
  const uint32_t stage0 = smem_u32(smem) + kCtlBytes;
  const uint32_t staging = stage0 + S * STAGE;                                    // kStagingBytes for each epilogue warp
  float* scales = reinterpret_cast<float*>(smem + kCtlBytes + S * STAGE + 8 * kStagingBytes);   // [2][2][BN]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_cta_rank() & 1, z = cluster_cta_rank() >> 1;
  volatile uint32_t* abort_word = &ctl->abort_word;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(smem_u32(&ctl->full[s]), 1);
      mbar_init(smem_u32(&ctl->empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&ctl->tmem_full[a]), 1);
      mbar_init(smem_u32(&ctl->tmem_empty[a]), 16);         // the epilogue warps of both CTAs
    }
    ctl->abort_word = 0;
    ctl->peer_lost = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&ctl->tmem_base), COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();                  // the partner's barriers exist before anything arrives on them
  tc_fence_after_sync();
  const uint32_t tmem_base = ctl->tmem_base;
  grid_dep_wait();
  grid_dep_launch();

  const int total = p.m_tiles * p.n_tiles, first = (int)blockIdx.x / (2 * Z), step = (int)gridDim.x / (2 * Z);
  const int kb0 = Z == 1 ? 0 : (int)((int64_t)p.KB * z / Z), kb1 = Z == 1 ? p.KB : (int)((int64_t)p.KB * (z + 1) / Z);
  if (warp == 0) {
    if (lane == 0) {
      prefetch_tensormap(&p.tmX);
      prefetch_tensormap(&p.tmW);
      int stage = 0;
      uint32_t phase = 0;
      int64_t issued = 0;
      bool ok = true;
      const int held = p.hold_back == (int)blockIdx.x ? kb1 - 1 : kb1;
      for (int w = first; w < total && ok; w += step) {
        int m, n;
        tile_of(w, p.m_tiles, p.n_tiles, m, n);
        const int t0 = m * 256 + (int)rank * 128, n0 = n * BN + (int)rank * (BN / 2);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(smem_u32(&ctl->empty[stage]), phase ^ 1, abort_word, 0x2100 + stage)) { ok = false; break; }
          const uint32_t st = stage0 + stage * STAGE, full = smem_u32(&ctl->full[stage]);
          if (rank == 0) mbar_expect_tx(full, 2 * STAGE);
          tma_load_2d_pair(st, &p.tmX, full, kb * kTileKI8, t0);
          if (kb < held) tma_load_2d_pair(st + kRowTileBytes, &p.tmW, full, kb * kTileKI8, n0);
          ++issued;
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
      }
      if (rank == 0 && (!ok || *abort_word)) drain_copies(ctl, issued, S);
    }
  } else if (warp == 1) {
    const uint32_t idesc = make_idesc_i8(256, BN);
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    for (int w = rank == 0 ? first : total; w < total && ok; w += step) {
      if (!mbar_wait(smem_u32(&ctl->tmem_empty[acc]), acc_phase ^ 1, abort_word, 0x2200 + acc)) break;
      tc_fence_after_sync();
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(smem_u32(&ctl->full[stage]), phase, abort_word, 0x2300 + stage)) { ok = false; break; }
        tc_fence_after_sync();
        __syncwarp();
        if (elect_one()) {
          const uint32_t st = stage0 + stage * STAGE;
          const uint32_t a_lo = desc_lo_sw(st), b_lo = desc_lo_sw(st + kRowTileBytes);
          const int steps = kb == p.KB - 1 ? p.k_tail_steps : 4;
#pragma unroll
          for (int s = 0; s < 4; ++s)
            if (s < steps) umma_i8<true>(tmem_base + acc * BN, a_lo + 2 * s, b_lo + 2 * s, idesc, (kb != kb0 || s != 0) ? 1u : 0u);
          commit_to_pair(smem_u32(&ctl->empty[stage]), z);
          if (kb == kb1 - 1) commit_to_pair(smem_u32(&ctl->tmem_full[acc]), z);
        }
        __syncwarp();
        if (++stage == S) { stage = 0; phase ^= 1; }
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
  }
  const int quad = warp & 3, half = (warp - 2) >> 2, te = (int)threadIdx.x - 64;
  const uint32_t rows_at = stage0 + (uint32_t)(quad * 32 + lane) * 16;    // Z > 1: [slot][column / 4][128 rows][4] int32
  // channel scales and biases of tile columns n0.. into buffer `acc`
  auto load_scales = [&](int n0, int acc) {
    float* sc = scales + acc * 2 * BN;
    for (int i = te; i < BN; i += 256) {
      const bool in = n0 + i < p.N;
      sc[i] = in ? p.w_scale[n0 + i] : 0.f;
      sc[BN + i] = (in && p.bias != nullptr) ? p.bias[n0 + i] : 0.f;
    }
  };
  bool ready = false;
  if constexpr (Z > 1) {
    // every product of the cluster is done before anything is written over its operands
    if (warp >= 2) {
      int m, n;
      tile_of(first, p.m_tiles, p.n_tiles, m, n);
      load_scales(n * BN, 0);
      ready = __all_sync(0xffffffffu, mbar_wait(smem_u32(&ctl->tmem_full[0]), 0, abort_word, 0x2400));
    }
    __syncwarp();
    tc_fence_before_sync();
    cluster_sync_all();
    tc_fence_after_sync();
    if (warp >= 2 && ready) {
      for (int d = 1; d < Z; ++d) {
        const uint32_t to = (z + d) % Z, slot = Z - 1 - d;               // the receiver counts its senders from behind
        const uint32_t dst = peer_smem(rows_at, 2 * to + rank) + slot * (BN / Z) * 512;
#pragma unroll 1
        for (int c = half * 16; c < BN / Z; c += 32) {
          uint32_t v[16];
          tmem_ld_32x32b_x16(tmem_base + ((uint32_t)(quad * 32) << 16) + to * (BN / Z) + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; i += 4) st_peer_v4(dst + (uint32_t)(c + i) * 512, v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      }
    }
    if (warp >= 2 && !ready && lane < 2 * Z) st_peer_u32(peer_smem(smem_u32(&ctl->peer_lost), (uint32_t)lane), 1);
    __syncwarp();
    cluster_sync_all();
    ready = ready && *(volatile uint32_t*)&ctl->peer_lost == 0;
  }
  if (warp >= 2) {
    const uint32_t mine = staging + (uint32_t)(warp - 2) * kStagingBytes;
    int acc = 0, w = first;
    uint32_t acc_phase = 0;
    const int first_col = Z > 1 ? (int)z * (BN / Z) : 0;
    for (; w < total; w += step) {
      int m, n;
      tile_of(w, p.m_tiles, p.n_tiles, m, n);
      const int row0 = m * 256 + (int)rank * 128 + quad * 32, n0 = n * BN;
      const float* sc = scales + acc * 2 * BN;
      if (Z == 1) load_scales(n0, acc);
      const float xs = row0 + lane < p.T ? p.x_scale[row0 + lane] : 0.f;
      const bool ok = Z > 1 ? ready : mbar_wait(smem_u32(&ctl->tmem_full[acc]), acc_phase, abort_word, 0x2400 + acc);
      uint32_t all;                        // every epilogue warp of the CTA sees the scales, or all of them give up
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                   : "=r"(all) : "r"((uint32_t)ok) : "memory");
      if (!all) break;
      tc_fence_after_sync();
      const uint32_t tacc = tmem_base + ((uint32_t)(quad * 32) << 16) + acc * BN;
#pragma unroll 1
      for (int c0 = first_col + half * kStoreCols; c0 < first_col + BN / Z; c0 += 2 * kStoreCols) {
        if (row0 >= p.T || n0 + c0 >= p.N) break;
        if (lane == 0) bulk_wait_read();    // the staging rows' previous copy has been read out
        __syncwarp();
#pragma unroll
        for (int h = 0; h < kStoreCols; h += 16) {
          uint32_t v[16];
          tmem_ld_32x32b_x16(tacc + c0 + h, v);
          tmem_ld_wait();
          if constexpr (Z > 1) {
#pragma unroll
            for (int slot = 0; slot < Z - 1; ++slot)
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const uint4 a = lds16(rows_at + (uint32_t)(slot * (BN / Z) + c0 - first_col + h + i) * 512);
                v[i] += a.x; v[i + 1] += a.y; v[i + 2] += a.z; v[i + 3] += a.w;
              }
          }
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const float4 ws = *reinterpret_cast<const float4*>(sc + c0 + h + i);
            const float4 bs = *reinterpret_cast<const float4*>(sc + BN + c0 + h + i);
            o[i / 2] = pack2(fmaf((float)(int)v[i] * xs, ws.x, bs.x), fmaf((float)(int)v[i + 1] * xs, ws.y, bs.y), p.fp16);
            o[i / 2 + 1] = pack2(fmaf((float)(int)v[i + 2] * xs, ws.z, bs.z), fmaf((float)(int)v[i + 3] * xs, ws.w, bs.w), p.fp16);
          }
          const uint32_t row = mine + (uint32_t)lane * 64, j = (uint32_t)h / 8, x = ((uint32_t)lane >> 1) & 3;    // 64-byte swizzle
          st_shared_v4(row + ((j ^ x) << 4), o[0], o[1], o[2], o[3]);
          st_shared_v4(row + (((j + 1) ^ x) << 4), o[4], o[5], o[6], o[7]);
        }
        if (p.store_tma) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&p.tmY, mine, n0 + c0, row0);
            bulk_commit();
          }
        } else {
          // rows of y that do not start on 16 bytes: two rows at a time, two neighbouring values a lane
          __syncwarp();
          const int col = n0 + c0 + (lane & 15) * 2;
          for (int r = lane >> 4; r < 32 && row0 + r < p.T; r += 2) {
            const uint32_t v = ld_shared_u32(mine + (uint32_t)r * 64 + (((((uint32_t)lane & 15) >> 2) ^ (((uint32_t)r >> 1) & 3)) << 4) + (lane & 3) * 4);
            uint16_t* dst = static_cast<uint16_t*>(p.y) + (int64_t)(row0 + r) * p.N + col;
            if (col < p.N) dst[0] = (uint16_t)v;
            if (col + 1 < p.N) dst[1] = (uint16_t)(v >> 16);
          }
          __syncwarp();
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(smem_u32(&ctl->tmem_empty[acc]));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (lane == 0) bulk_wait_all();
    // A wait ran out: the tiles that are left become NaN, as a row that cannot be quantised does.
    for (; w < total; w += step) {
      int m, n;
      tile_of(w, p.m_tiles, p.n_tiles, m, n);
      const int row0 = m * 256 + (int)rank * 128 + quad * 32;
      for (int r = row0; r < min(row0 + 32, p.T); ++r)
        for (int c = n * BN + first_col + half * 32 + lane; c < min(n * BN + first_col + BN / Z, p.N); c += 64)
          static_cast<uint16_t*>(p.y)[(int64_t)r * p.N + c] = p.fp16 ? 0x7e00 : 0x7fc0;
    }
  }

  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (threadIdx.x == 0 && ctl->abort_word != 0) report_abort(p, ctl->abort_word);
  cluster_sync_all();     // neither CTA leaves while the other's products or arrivals may still touch it
  if (warp == 1) tmem_dealloc_pair(tmem_base, COLS);
}

// ------------------------------------------------------------------------------------ host
int encode_rows(CUtensorMap* map, const void* base, int K, int rows, int box_rows, const char* what) {
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)K};
  cuuint32_t box[2] = {kTileKI8, (cuuint32_t)box_rows};
  return encode_map_sw(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, what);
}

struct Variant {
  bool pair, fused;
  int tokens, splits, stages;    // split
  int bn, z;                     // pair: features of a tile, pairs that share K
};

Variant pick_variant(int T, int N, int K, int force, bool quantise) {
  const int KB = (K + kTileKI8 - 1) / kTileKI8;
  Variant v = {};
  const int sms = device_sm_count();
  v.pair = force == 2 || (force == 0 && T > 64);      // T = 64: 9.8 against 10.8 us; T = 128: 12.6 against 10.9 (4096 x 4096, the only N x K measured)
  if (v.pair) {
    // Cost of a tile shape in us, fitted to calls of one round (T = 256 to 1000, N = 2048 and 4096, K = 4096 and 7168): rounds
    // of tiles over the pairs x k-blocks x what one takes, 0.30 for 256 features and 0.216 for 128; what a call does not
    // overlap, 7.0 and 6.3; joining two halves of K, 2.3 and 1.3.
    const int pairs = sms / 2, mt = (T + 255) / 256;
    double best = 0;
    for (int bn : {256, 128})
      for (int z : {1, 2}) {
        const int64_t tiles = (int64_t)mt * ((N + bn - 1) / bn);
        if (z > 1 && (tiles * z > pairs || KB < 4 * z)) continue;
        const double rounds = z > 1 ? 1.0 : (double)((tiles + pairs - 1) / pairs);
        const double cost = rounds * ((KB + z - 1) / z) * (bn == 256 ? 0.30 : 0.216) + (bn == 256 ? 7.0 : 6.3) +
                            (z == 1 ? 0.0 : bn == 256 ? 2.3 : 1.3);
        if (v.bn == 0 || cost < best) { best = cost; v.bn = bn; v.z = z; }
      }
    return v;
  }
  v.tokens = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : kMaxTokenTile;
  const int64_t tiles = (int64_t)((N + kRowTile - 1) / kRowTile) * ((T + v.tokens - 1) / v.tokens);
  v.splits = 1;
  while (v.splits < 8 && tiles * v.splits * 2 <= 3 * sms && KB / (v.splits * 2) >= 2) v.splits *= 2;
  const int kb = (KB + v.splits - 1) / v.splits;
  v.fused = quantise && T == 1 && kb <= kFusedBlocks;
  const int stage = kRowTileBytes + (v.fused ? 0 : v.tokens * kTileKI8);
  v.stages = std::min({kb, kMaxStagesI8, (110 * 1024 - (v.fused ? kb * kFusedBlockBytes : 0)) / stage});      // two CTAs to an SM
  return v;
}

}  // namespace

struct LinearArgs {
  const void* x; int x_dtype;                          // rows; int8 ones with q = x and their scale
  const void* q; const float* x_scale;
  const void* w; const float* w_scale; const float* bias;
  void* y;
  int T, N, K, fp16, early_weights;
  int32_t* status;
  bool hold_back;
};
int launch_linear_int8(const LinearArgs& a, const Variant& v, cudaStream_t st) {
  LinearParams p;
  memset(&p, 0, sizeof(p));
  const int T = a.T, N = a.N, K = a.K;
  p.K = K;
  p.KB = (K + kTileKI8 - 1) / kTileKI8;
  p.k_tail_steps = (K - (p.KB - 1) * kTileKI8 + 31) / 32;
  p.T = T; p.N = N; p.x_scale = a.x_scale; p.w_scale = a.w_scale; p.bias = a.bias; p.y = a.y; p.status = a.status; p.fp16 = a.fp16;
  p.hold_back = a.hold_back ? (v.pair ? 1 : 0) : -1;      // of a pair, the CTA that does not issue the products
  if (!v.pair) {
    B200_CHECK_ARG(v.tokens <= kMaxTokenTile, "linear_int8: token tile %d", v.tokens);
    p.tokens = v.tokens; p.splits = v.splits; p.stages = v.stages; p.early_weights = a.early_weights;
    p.x = a.x; p.x_dtype = a.x_dtype;
    p.x_vec = ((uintptr_t)a.x & 15) == 0;
    if (!v.fused)
      if (int rc = encode_rows(&p.tmX, a.q, K, T, v.tokens, "int8 token rows")) return rc;
    if (int rc = encode_rows(&p.tmW, a.w, K, N, kRowTile, "int8 weights")) return rc;
    const int n_tiles = (N + kRowTile - 1) / kRowTile, t_tiles = (T + v.tokens - 1) / v.tokens;
    B200_CHECK_ARG(t_tiles <= 65535, "linear_int8: %d tokens", T);
    const int stage = kRowTileBytes + (v.fused ? 0 : v.tokens * kTileKI8);
    const int blocks = v.fused ? ((p.KB + v.splits - 1) / v.splits) * kFusedBlockBytes : 0;
    // At least the share of shared memory that its columns are of tensor memory, and 64 KB, which leaves no room beside a CTA that
    // takes all columns: a CTA that fits an SM finds its columns there instead of blocking in their allocation.  (It waits for no
    // other CTA while it holds them.  The pair kernel's CTAs do; they leave 13 KB of an SM, too little for another such kernel.)
    const int share = std::max((int)((int64_t)kSmemLimitI8 * std::max(32, v.tokens) / 512), 64 * 1024);
    const int bytes = std::max({v.stages * stage + blocks, std::min(v.tokens, T) * kRowTile * 4 + 16 * kRowTile * 4, share});
    const size_t smem = 1024 + kCtlBytes + (size_t)bytes;
    void (*k)(LinearParams) = v.fused ? linear_int8_split_kernel<true> : linear_int8_split_kernel<false>;
    B200_CHECK_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimitI8 - 1024));
    B200_CHECK_CUDA(launch_chained_cluster(k, dim3(n_tiles * v.splits, t_tiles), dim3(kThreadsI8), smem, st, v.splits, p));
    return 0;
  }
  const int bn = v.bn;
  p.m_tiles = (T + 255) / 256;
  p.n_tiles = (N + bn - 1) / bn;
  if (int rc = encode_rows(&p.tmX, a.q, K, T, 128, "int8 token rows")) return rc;
  if (int rc = encode_rows(&p.tmW, a.w, K, N, bn / 2, "int8 weights")) return rc;
  p.store_tma = N % 8 == 0 && ((uintptr_t)a.y & 15) == 0;
  if (p.store_tma) {
    cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)T};
    cuuint64_t strides[1] = {(cuuint64_t)N * 2};
    cuuint32_t box[2] = {kStoreCols, 32};
    if (int rc = encode_map_sw(&p.tmY, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, a.y, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B,
                               CU_TENSOR_MAP_L2_PROMOTION_NONE, "linear output"))
      return rc;
  }
  const int stage = kRowTileBytes + bn / 2 * kTileKI8;
  p.stages = std::min((kSmemLimitI8 - 1024 - kCtlBytes - 8 * kStagingBytes - kPairScaleBytes) / stage, kMaxStagesI8);
  const size_t smem = 1024 + kCtlBytes + (size_t)p.stages * stage + 8 * kStagingBytes + kPairScaleBytes;
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
  B200_CHECK_ARG(tiles < (1ll << 30), "linear_int8: T=%d N=%d", T, N);
  const int grid = 2 * v.z * (v.z > 1 ? (int)tiles : (int)std::min<int64_t>(device_sm_count() / 2, tiles));
  void (*k)(LinearParams) = bn == 256 ? (v.z == 2 ? linear_int8_pair_kernel<256, 2> : linear_int8_pair_kernel<256, 1>)
                                      : (v.z == 2 ? linear_int8_pair_kernel<128, 2> : linear_int8_pair_kernel<128, 1>);
  B200_CHECK_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimitI8));
  B200_CHECK_CUDA(launch_chained_cluster(k, dim3(grid), dim3(kPairThreads), smem, st, 2 * v.z, p));
  return 0;
}

}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_linear_int8_status(int32_t* status2) {
  B200_CHECK_ARG(status2 != nullptr, "linear_int8_status: NULL pointer");
  B200_CHECK_CUDA(cudaDeviceSynchronize());
  B200_CHECK_CUDA(cudaMemcpyFromSymbol(status2, g_linear_status, 2 * sizeof(int32_t)));
  return 0;
}

extern "C" int b200moe_linear_int8_workspace(int32_t T, int32_t N, int32_t K, int32_t variant, int64_t* bytes) {
  variant &= ~B200MOE_LINEAR_HOLD_BACK;
  B200_CHECK_ARG(bytes != nullptr && T >= 0 && N >= 1 && K >= 1 && variant >= 0 && variant <= 2, "linear_int8_workspace: T=%d N=%d K=%d", T, N, K);
  const Variant v = pick_variant(T, N, K, variant, true);
  *bytes = T == 0 || v.fused ? 0 : round_up64((int64_t)T * K, 256) + (int64_t)T * 4;     // the quantised rows and their scales
  return 0;
}

extern "C" int b200moe_linear_int8(const void* x, int64_t x_stride, int32_t x_dtype, const float* x_scale, const void* weight,
                                   const float* weight_scale, const float* bias, int32_t T, int32_t N, int32_t K, int32_t out_dtype,
                                   int32_t variant, void* workspace, int64_t workspace_bytes, int32_t* status, void* y, void* stream) {
  B200_CHECK_ARG(T >= 0 && N >= 1 && K >= 16 && K % 16 == 0 && K < (1 << 17), "linear_int8: T=%d N=%d K=%d (K a multiple of 16 below 2^17)",
                 T, N, K);
  B200_CHECK_ARG(out_dtype == B200MOE_T_BF16 || out_dtype == B200MOE_T_FP16, "linear_int8: out dtype %d", out_dtype);
  B200_CHECK_ARG(x_dtype == B200MOE_T_INT8 || (x_dtype >= B200MOE_T_BF16 && x_dtype <= B200MOE_T_FP32), "linear_int8: x dtype %d", x_dtype);
  const bool hold_back = (variant & B200MOE_LINEAR_HOLD_BACK) != 0;
  variant &= ~B200MOE_LINEAR_HOLD_BACK;
  B200_CHECK_ARG(variant >= 0 && variant <= 2, "linear_int8: variant %d", variant);
  if (T == 0) return 0;
  B200_CHECK_ARG(x && weight && weight_scale && y, "linear_int8: NULL pointer");
  B200_CHECK_ARG(((uintptr_t)weight & 15) == 0, "linear_int8: weight must be 16-byte aligned");
  B200_CHECK_ARG(((uintptr_t)y & 7) == 0, "linear_int8: y must be 8-byte aligned");
  cudaStream_t st = (cudaStream_t)stream;
  const bool quantise = x_dtype != B200MOE_T_INT8;
  const Variant v = pick_variant(T, N, K, variant, quantise);
  LinearArgs a = {x, x_dtype, x, x_scale, weight, weight_scale, bias, y, T, N, K, out_dtype == B200MOE_T_FP16, quantise, status, hold_back};
  if (!quantise) {
    B200_CHECK_ARG(x_scale != nullptr && x_stride == K && ((uintptr_t)x & 15) == 0, "linear_int8: 8-bit rows must be contiguous, 16-byte aligned and have x_scale");
  } else {
    B200_CHECK_ARG(K <= 16384 && x_stride >= 0, "linear_int8: rows of %d values, %lld apart", K, (long long)x_stride);
    if (!v.fused) {
      const int64_t rows = round_up64((int64_t)T * K, 256);
      B200_CHECK_ARG(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= rows + (int64_t)T * 4,
                     "linear_int8: workspace holds %lld bytes of %lld", (long long)workspace_bytes, (long long)(rows + (int64_t)T * 4));
      float* scale = (float*)((uint8_t*)workspace + rows);
      if (int rc = b200moe_quantize_int8(x, x_stride, T, K, x_dtype, workspace, scale, stream)) return rc;
      a.q = workspace;
      a.x_scale = scale;
    }
  }
  return launch_linear_int8(a, v, st);
}
