// Tensor-core products of the block-scaled 8-bit arithmetic (formats and definition: fp8.cu).
//
// tcgen05 kind::f8f6f4 multiplies a block of 128 columns at a time into tensor memory; the weight's
// scale is a general float32 per block, so the block sums cannot stay there: the epilogue warps read
// each one out, scale it and add it to float32 sums in their registers while the next block is
// multiplied into the other half of tensor memory.
//
//   rows on the MMA's 128 lanes (fp8_rows_kernel)      many rows: tiles of 128 rows x 256 weight rows;
//       a thread owns a row and 128 of its columns, so a block costs it one scale and 128 FMAs.
//   weights on the lanes (fp8_weights_kernel)          few rows: tiles of 128 weight rows x 16..128
//       rows, the K blocks of a tile split over a cluster of up to eight CTAs, whose sums meet in
//       shared memory.  Bound by the weight bytes, so what counts is that every SM streams.
//
// Each in two forms: the plain product, and gate / up with the SwiGLU and the next quantisation in the
// epilogue (both matrices in one tile, so that a thread meets gate and up of the same feature).
#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "fp8.cuh"
#include "internal.h"
#include "tc_ptx.cuh"

namespace glmrt {
namespace {

using namespace tc;

__device__ uint32_t g_fp8_error;       // kErrWaitTimeout when a bounded wait ran out (glmrt_b200_fp8_check)

__device__ __forceinline__ void tc_mma_fp8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// E4M3 x E4M3 -> float32, both operands K-major, M = 128, N = n.
__device__ __forceinline__ uint32_t idesc_fp8(uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((128u >> 4) << 24); }

constexpr int kTileBytes = 128 * kFp8Block;            // 128 rows of one K block

// ---------------------------------------------------------------------------------------------------
// Many rows
// ---------------------------------------------------------------------------------------------------
constexpr int kRowsStages = 4;
constexpr int kRowsEpiWarps = 8;
constexpr int kRowsThreads = 32 * (2 + kRowsEpiWarps);
constexpr int kRowsN = 256;
constexpr int kRowsStageBytes = kTileBytes + 2 * kTileBytes;
constexpr size_t kRowsSmem = static_cast<size_t>(kRowsStages) * kRowsStageBytes + 1024 + 256 + 128 * 2 * 4;

struct RowsArgs {
  const float* xs;            // [blocks][xs_stride]
  const float *ws0, *ws1;     // weight scales (gate / up: both)
  void* out;                  // product: [rows, n] bf16 or float32; SwiGLU: codes [rows, n]
  float* out_scales;          // SwiGLU: [ceil(n / 128)][out_stride]
  int rows, n, k, xs_stride, out_stride;
  int vector_out;             // rows of the output start on 16-byte boundaries
};

// kMode 0: bf16 product, 1: float32 product, 2: SwiGLU of gate / up, quantised
template <int kMode>
__global__ void __launch_bounds__(kRowsThreads, 1)
fp8_rows_kernel(RowsArgs a, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w0,
                const __grid_constant__ CUtensorMap map_w1) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + static_cast<size_t>(kRowsStages) * kRowsStageBytes);
  uint64_t* empty_bar = full_bar + kRowsStages;
  uint64_t* acc_full = empty_bar + kRowsStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  float* amax_x = reinterpret_cast<float*>(smem + static_cast<size_t>(kRowsStages) * kRowsStageBytes + 256);   // [2][128]

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int blocks = (a.k + kFp8Block - 1) / kFp8Block;
  const int per_tile = kMode == 2 ? 128 : kRowsN;                 // output columns of a tile
  const int n_tiles = (a.n + per_tile - 1) / per_tile, m_tiles = (a.rows + 127) / 128;
  const int tiles = n_tiles * m_tiles;

  if (threadIdx.x == 32) {
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w0);
    if (kMode == 2) prefetch_tensormap(&map_w1);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kRowsStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kRowsEpiWarps);
    }
    *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();      // after the wait: a successor may then rely on everything before this kernel

  // tiles of one column of weight tiles follow each other, so that the rows stay in L2 and the weights are read once
  auto tile_m = [&](int tile) { return tile % m_tiles; };
  auto tile_n = [&](int tile) { return tile / m_tiles; };

  if (warp == 0) {
    const uint64_t pol = policy_evict_last();
    int stage = 0;
    uint32_t phase = 0;
    bool alive = true;
    for (int tile = blockIdx.x; tile < tiles && alive; tile += gridDim.x) {
      const int m0 = tile_m(tile) * 128, n0 = tile_n(tile) * per_tile;
      for (int b = 0; b < blocks; ++b) {
        if (!mbar_wait_warp(&empty_bar[stage], phase ^ 1u, abort_flag)) { alive = false; break; }
        if (elect_one()) {
          const uint32_t s_a = smem_u32(smem + static_cast<size_t>(stage) * kRowsStageBytes), s_b = s_a + kTileBytes;
          mbar_expect_tx(&full_bar[stage], kRowsStageBytes);
          tma_load_2d(s_a, &map_x, &full_bar[stage], b * kFp8Block, m0, pol);
          if (kMode == 2) {
            // 64 gate rows, the 64 up rows of the same features, and the same for the next 64
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              tma_load_2d(s_b + h * kTileBytes, &map_w0, &full_bar[stage], b * kFp8Block, n0 + 64 * h, pol);
              tma_load_2d(s_b + h * kTileBytes + kTileBytes / 2, &map_w1, &full_bar[stage], b * kFp8Block, n0 + 64 * h, pol);
            }
          } else {
            tma_load_2d(s_b, &map_w0, &full_bar[stage], b * kFp8Block, n0, pol);
          }
        }
        __syncwarp();
        if (++stage == kRowsStages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    int stage = 0, abuf = 0;
    uint32_t phase = 0, aphase = 0;
    bool alive = true;
    const uint32_t idesc = idesc_fp8(kRowsN);
    for (int tile = blockIdx.x; tile < tiles && alive; tile += gridDim.x) {
      for (int b = 0; b < blocks; ++b) {
        if (!mbar_wait_warp(&acc_empty[abuf], aphase ^ 1u, abort_flag) ||
            !mbar_wait_warp(&full_bar[stage], phase, abort_flag)) { alive = false; break; }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t s_a = smem_u32(smem + static_cast<size_t>(stage) * kRowsStageBytes), s_b = s_a + kTileBytes;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc_mma_fp8(tmem_base + abuf * kRowsN, desc_sw128(s_a + kk * 32), desc_sw128(s_b + kk * 32), idesc, kk != 0 ? 1u : 0u);
          tc_commit(&empty_bar[stage]);
          tc_commit(&acc_full[abuf]);
        }
        __syncwarp();
        if (++stage == kRowsStages) { stage = 0; phase ^= 1u; }
        abuf ^= 1;
        if (abuf == 0) aphase ^= 1u;
      }
    }
  } else {
    const int quad = warp & 3, part = (warp - 2) >> 2;       // tensor-memory lanes, half of the tile's columns
    const int lane_row = quad * 32 + lane;
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + part * 128;
    int abuf = 0;
    uint32_t aphase = 0;
    // A warp whose wait ran out keeps step with the others (they meet at barriers), computing nothing valid.
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      const int row = tile_m(tile) * 128 + lane_row, n0 = tile_n(tile) * per_tile;
      // the product's halves are two weight blocks; gate and up share the block number of their features
      const int wb = kMode == 2 ? tile_n(tile) : min(tile_n(tile) * 2 + part, (a.n - 1) / kFp8Block);
      const float* xs = a.xs + row;                          // padded to whole tiles
      const float* ws0 = a.ws0 + static_cast<size_t>(wb) * blocks;
      const float* ws1 = kMode == 2 ? a.ws1 + static_cast<size_t>(wb) * blocks : nullptr;
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
      for (int b = 0; b < blocks; ++b) {
        const float sx = __ldg(xs + static_cast<size_t>(b) * a.xs_stride);
        const float s0 = sx * __ldg(ws0 + b), s1 = kMode == 2 ? sx * __ldg(ws1 + b) : s0;
        mbar_wait_warp(&acc_full[abuf], aphase, abort_flag);
        tc_fence_after();
        const uint32_t t = t_lane + abuf * kRowsN;
        uint32_t v[2][16];
        tc_load16(t, v[0]);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          tc_wait_ld();
          if (c < 7) tc_load16(t + (c + 1) * 16, v[(c + 1) & 1]);
          const float s = kMode == 2 && c >= 4 ? s1 : s0;
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[c * 16 + i] = fmaf(__uint_as_float(v[c & 1][i]), s, acc[c * 16 + i]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[abuf]);
        abuf ^= 1;
        if (abuf == 0) aphase ^= 1u;
      }
      if (kMode == 2) {
        // features n0 + 64 part .. + 63: gate in acc[0..63], up in acc[64..127]
        uint32_t amax = 0u;
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          acc[i] = fp8_swiglu(acc[i], acc[64 + i]);
          amax = max(amax, __float_as_uint(acc[i]) & 0x7fffffffu);
        }
        amax_x[part * 128 + lane_row] = __uint_as_float(amax);
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kRowsEpiWarps) : "memory");
        amax = max(amax, __float_as_uint(amax_x[(part ^ 1) * 128 + lane_row]));
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kRowsEpiWarps) : "memory");   // read before the next tile writes
        float inv;
        const float scale = fp8_block_scale(amax, &inv);
        if (row < a.rows) {
          if (part == 0) a.out_scales[static_cast<size_t>(wb) * a.out_stride + row] = scale;
          uint8_t* dst = static_cast<uint8_t*>(a.out) + static_cast<size_t>(row) * a.n + n0 + 64 * part;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint4 q;
            q.x = fp8_pack4(acc[16 * c] * inv, acc[16 * c + 1] * inv, acc[16 * c + 2] * inv, acc[16 * c + 3] * inv);
            q.y = fp8_pack4(acc[16 * c + 4] * inv, acc[16 * c + 5] * inv, acc[16 * c + 6] * inv, acc[16 * c + 7] * inv);
            q.z = fp8_pack4(acc[16 * c + 8] * inv, acc[16 * c + 9] * inv, acc[16 * c + 10] * inv, acc[16 * c + 11] * inv);
            q.w = fp8_pack4(acc[16 * c + 12] * inv, acc[16 * c + 13] * inv, acc[16 * c + 14] * inv, acc[16 * c + 15] * inv);
            if (n0 + 64 * part + 16 * c < a.n) *reinterpret_cast<uint4*>(dst + 16 * c) = q;      // n % 16 == 0
          }
        }
      } else if (row < a.rows) {
        const int c0 = n0 + 128 * part;
        constexpr int kPer = kMode == 0 ? 8 : 4;             // values of 16 bytes
#pragma unroll
        for (int c = 0; c < 128; c += kPer) {
          if (c0 + c >= a.n) continue;
          if (a.vector_out) {                                // n is a multiple of kPer
            uint4 q;
            if constexpr (kMode == 0) {
              q.x = pack_bf16x2(acc[c], acc[c + 1]); q.y = pack_bf16x2(acc[c + 2], acc[c + 3]);
              q.z = pack_bf16x2(acc[c + 4], acc[c + 5]); q.w = pack_bf16x2(acc[c + 6], acc[c + 7]);
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + static_cast<size_t>(row) * a.n + c0 + c) = q;
            } else {
              *reinterpret_cast<float4*>(static_cast<float*>(a.out) + static_cast<size_t>(row) * a.n + c0 + c) =
                  make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
              if (c0 + c + i < a.n) {
                if constexpr (kMode == 0) fp8_store(static_cast<uint16_t*>(a.out) + static_cast<size_t>(row) * a.n + c0 + c + i, acc[c + i]);
                else fp8_store(static_cast<float*>(a.out) + static_cast<size_t>(row) * a.n + c0 + c + i, acc[c + i]);
              }
          }
        }
      }
    }
  }

  if (*abort_flag != 0u) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);   // let copies in flight land
    if (threadIdx.x == 0) atomicOr(&g_fp8_error, static_cast<uint32_t>(kErrWaitTimeout));
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, 512);
}

// ---------------------------------------------------------------------------------------------------
// Few rows
// ---------------------------------------------------------------------------------------------------
struct WeightsArgs {
  const float* xs;            // [blocks][xs_stride]
  const float *ws0, *ws1;
  void* out;
  float* out_scales;
  int rows, n, k, xs_stride, out_stride;
};

template <int kMode, int kN>
struct WCfg {
  static constexpr int kMats = kMode == 2 ? 2 : 1;
  static constexpr int kStageBytes = kMats * kTileBytes + kN * kFp8Block;
  static constexpr int kStages = 184320 / kStageBytes < 10 ? 184320 / kStageBytes : 10;
  static constexpr int kAccCols = kMats * kN;                       // of one block
  static constexpr int kTmemCols = 2 * kAccCols < 32 ? 32 : 2 * kAccCols;
  static constexpr int kThreads = 192;
  static constexpr size_t kSmem = static_cast<size_t>(kStages) * kStageBytes + 1024 + 512 + 4 * kN * 4;
  static_assert(static_cast<size_t>(kStages) * kStageBytes >= static_cast<size_t>(kMats + 1) * kN * 128 * 4, "partial sums and the activation reuse the ring");
};

// grid (weight tiles, splits, row tiles), cluster (1, splits, 1).
template <int kMode, int kN>
__global__ void __launch_bounds__(WCfg<kMode, kN>::kThreads, 1)
fp8_weights_kernel(WeightsArgs a, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w0,
                   const __grid_constant__ CUtensorMap map_w1) {
  using C = WCfg<kMode, kN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + static_cast<size_t>(C::kStages) * C::kStageBytes);
  uint64_t* empty_bar = full_bar + C::kStages;
  uint64_t* acc_full = empty_bar + C::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  uint32_t* amax_x = reinterpret_cast<uint32_t*>(smem + static_cast<size_t>(C::kStages) * C::kStageBytes + 512);   // [4][kN]

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int blocks = (a.k + kFp8Block - 1) / kFp8Block;
  const int splits = gridDim.y, split = blockIdx.y;
  const int b0 = blocks * split / splits, b1 = blocks * (split + 1) / splits;
  const int w0 = blockIdx.x * 128, m0 = blockIdx.z * kN;

  if (threadIdx.x == 32) {
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w0);
    if (kMode == 2) prefetch_tensormap(&map_w1);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4);
    }
    *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (warp == 1) tmem_alloc(tmem_slot, C::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // The weights do not come from the previous kernel, and that kernel let this one start only after everything
    // before it had finished: the first stages' weights are asked for before its rows are waited for.
    const uint64_t pol = policy_evict_first();
    auto load_w = [&](int stage, int b) {
      const uint32_t s_a = smem_u32(smem + static_cast<size_t>(stage) * C::kStageBytes);
      mbar_expect_tx(&full_bar[stage], C::kStageBytes);
      tma_load_2d(s_a, &map_w0, &full_bar[stage], b * kFp8Block, w0, pol);
      if (kMode == 2) tma_load_2d(s_a + kTileBytes, &map_w1, &full_bar[stage], b * kFp8Block, w0, pol);
    };
    auto load_x = [&](int stage, int b) {
      tma_load_2d(smem_u32(smem + static_cast<size_t>(stage) * C::kStageBytes) + C::kMats * kTileBytes, &map_x, &full_bar[stage],
                  b * kFp8Block, m0, policy_evict_last());
    };
    const int ahead = min(C::kStages, b1 - b0);
    if (elect_one())
      for (int i = 0; i < ahead; ++i) load_w(i, b0 + i);
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();
    if (elect_one())
      for (int i = 0; i < ahead; ++i) load_x(i, b0 + i);
    __syncwarp();
    int stage = 0;
    uint32_t phase = 0;
    for (int b = b0 + ahead; b < b1; ++b) {
      if (!mbar_wait_warp(&empty_bar[stage], phase, abort_flag)) break;
      if (elect_one()) {
        load_w(stage, b);
        load_x(stage, b);
      }
      __syncwarp();
      if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
    }
  } else if (warp == 1) {
    pdl_wait();
    int stage = 0, abuf = 0;
    uint32_t phase = 0, aphase = 0;
    const uint32_t idesc = idesc_fp8(kN);
    for (int b = b0; b < b1; ++b) {
      if (!mbar_wait_warp(&acc_empty[abuf], aphase ^ 1u, abort_flag) ||
          !mbar_wait_warp(&full_bar[stage], phase, abort_flag)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t s_a = smem_u32(smem + static_cast<size_t>(stage) * C::kStageBytes), s_x = s_a + C::kMats * kTileBytes;
#pragma unroll
        for (int mat = 0; mat < C::kMats; ++mat)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc_mma_fp8(tmem_base + abuf * C::kAccCols + mat * kN, desc_sw128(s_a + mat * kTileBytes + kk * 32),
                       desc_sw128(s_x + kk * 32), idesc, kk != 0 ? 1u : 0u);
        tc_commit(&empty_bar[stage]);
        tc_commit(&acc_full[abuf]);
      }
      __syncwarp();
      if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
      abuf ^= 1;
      if (abuf == 0) aphase ^= 1u;
    }
  }
  const int quad = warp & 3, lane_row = quad * 32 + lane;           // epilogue warps: weight row of the tile
  float acc[C::kMats][kN];
  if (warp >= 2) {
    pdl_wait();
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
    const size_t wb = static_cast<size_t>(blockIdx.x) * blocks;
#pragma unroll
    for (int mat = 0; mat < C::kMats; ++mat)
#pragma unroll
      for (int j = 0; j < kN; ++j) acc[mat][j] = 0.0f;
    int abuf = 0;
    uint32_t aphase = 0;
    for (int b = b0; b < b1; ++b) {
      const float* xs = a.xs + static_cast<size_t>(b) * a.xs_stride + m0;       // padded to whole tiles of 128
      const float sw[2] = {__ldg(a.ws0 + wb + b), kMode == 2 ? __ldg(a.ws1 + wb + b) : 0.0f};
      if (!mbar_wait_warp(&acc_full[abuf], aphase, abort_flag)) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kN / 16; ++c) {
        float sx[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 q = *reinterpret_cast<const float4*>(xs + c * 16 + i * 4);
          sx[4 * i] = q.x; sx[4 * i + 1] = q.y; sx[4 * i + 2] = q.z; sx[4 * i + 3] = q.w;
        }
#pragma unroll
        for (int mat = 0; mat < C::kMats; ++mat) {
          uint32_t v[16];
          tc_load16(t_lane + abuf * C::kAccCols + mat * kN + c * 16, v);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            acc[mat][c * 16 + i] = fmaf(__uint_as_float(v[i]), sx[i] * sw[mat], acc[mat][c * 16 + i]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[abuf]);
      abuf ^= 1;
      if (abuf == 0) aphase ^= 1u;
    }
  }

  // ---- the splits' sums meet: [matrix][row of x][weight row] in each CTA's ring, whose copies have all been used ----
  __syncthreads();
  if (*abort_flag != 0u) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);   // let copies in flight land
    if (threadIdx.x == 0) atomicOr(&g_fp8_error, static_cast<uint32_t>(kErrWaitTimeout));
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, C::kTmemCols);
  float* part = reinterpret_cast<float*>(smem);
  if (splits > 1) {
    if (warp >= 2)
#pragma unroll
      for (int mat = 0; mat < C::kMats; ++mat)
#pragma unroll
        for (int j = 0; j < kN; ++j) part[(mat * kN + j) * 128 + lane_row] = acc[mat][j];
    cluster_sync_all();
  }
  // this CTA finishes rows j0 .. j1 of the tile, the splits added in order
  const int valid = min(kN, a.rows - m0);
  const int j0 = valid * split / splits, j1 = valid * (split + 1) / splits;
  const int feature = w0 + lane_row;
  if (warp >= 2) {
    const uint32_t part_at = smem_u32(part);
    auto total = [&](int mat, int j) {
      float v[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        v[r] = 0.0f;
        if (r < splits)
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[r]) : "r"(cluster_addr(part_at + ((mat * kN + j) * 128 + lane_row) * 4, r)) : "memory");
      }
      float s = v[0];
#pragma unroll
      for (int r = 1; r < 8; ++r) s += v[r];
      return s;
    };
    if constexpr (kMode != 2) {
      if (splits == 1) {
#pragma unroll
        for (int j = 0; j < kN; ++j)
          if (j < valid && feature < a.n) {
            if constexpr (kMode == 0) fp8_store(static_cast<uint16_t*>(a.out) + static_cast<size_t>(m0 + j) * a.n + feature, acc[0][j]);
            else fp8_store(static_cast<float*>(a.out) + static_cast<size_t>(m0 + j) * a.n + feature, acc[0][j]);
          }
      } else {
        for (int j = j0; j < j1; ++j) {
          const float y = total(0, j);
          if (feature < a.n) {
            if constexpr (kMode == 0) fp8_store(static_cast<uint16_t*>(a.out) + static_cast<size_t>(m0 + j) * a.n + feature, y);
            else fp8_store(static_cast<float*>(a.out) + static_cast<size_t>(m0 + j) * a.n + feature, y);
          }
        }
      }
    } else {
      // SwiGLU, then the block's (128 features of one row) largest magnitude over the four warps
      float* act = part + C::kMats * kN * 128;              // [row of x][feature], behind the partial sums
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        if (j < j0 || j >= j1) continue;
        const float v = splits == 1 ? fp8_swiglu(acc[0][j], acc[C::kMats - 1][j]) : fp8_swiglu(total(0, j), total(1, j));
        act[j * 128 + lane_row] = v;
        const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu);
        if (lane == 0) amax_x[quad * kN + j] = m;
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      for (int j = j0; j < j1; ++j) {
        const float v = act[j * 128 + lane_row];
        const uint32_t m = max(max(amax_x[j], amax_x[kN + j]), max(amax_x[2 * kN + j], amax_x[3 * kN + j]));
        float inv;
        const float scale = fp8_block_scale(m, &inv);
        const size_t row = static_cast<size_t>(m0 + j);
        if (feature < a.n) static_cast<uint8_t*>(a.out)[row * a.n + feature] =
            static_cast<uint8_t>(__nv_cvt_float_to_fp8(v * inv, __NV_SATFINITE, __NV_E4M3));
        if (lane_row == 0) a.out_scales[static_cast<size_t>(blockIdx.x) * a.out_stride + row] = scale;
      }
    }
  }
  if (splits > 1) cluster_sync_all();       // nobody leaves while its sums may still be read
}

template <int kMode, int kN>
glmrt_status_t launch_weights(const Fp8Gemm& g, int splits, cudaStream_t s) {
  using C = WCfg<kMode, kN>;
  CUtensorMap mx, m0, m1;
  GLMRT_RETURN_IF_ERROR(make_bytes_tensor_map(&mx, g.x, g.rows, g.k, kN));
  GLMRT_RETURN_IF_ERROR(make_bytes_tensor_map(&m0, g.w0, g.n, g.k, 128));
  if (kMode == 2) GLMRT_RETURN_IF_ERROR(make_bytes_tensor_map(&m1, g.w1, g.n, g.k, 128));
  else m1 = m0;
  WeightsArgs a{g.xs, g.ws0, g.ws1, g.out, g.out_scales, g.rows, g.n, g.k, g.xs_stride, g.out_stride};
  static std::atomic<uint64_t> configured{0};
  GLMRT_RETURN_IF_ERROR(ensure_smem_limit(configured, fp8_weights_kernel<kMode, kN>, C::kSmem, "cudaFuncSetAttribute(fp8_weights_kernel)"));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((g.n + 127) / 128), static_cast<unsigned>(splits), static_cast<unsigned>((g.rows + kN - 1) / kN));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1; attr[0].val.clusterDim.y = static_cast<unsigned>(splits); attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t err = cudaLaunchKernelEx(&cfg, fp8_weights_kernel<kMode, kN>, a, mx, m0, m1);
  if (err != cudaSuccess) return fail_cuda(GLMRT_STATUS_COPY_FAILED, "fp8_weights_kernel", err);
  GLMRT_LAUNCH_CHECK("fp8_weights_kernel");
  return GLMRT_STATUS_OK;
}

template <int kMode>
glmrt_status_t launch_rows(const Fp8Gemm& g, int sm_count, cudaStream_t s) {
  CUtensorMap mx, m0, m1;
  GLMRT_RETURN_IF_ERROR(make_bytes_tensor_map(&mx, g.x, g.rows, g.k, 128));
  GLMRT_RETURN_IF_ERROR(make_bytes_tensor_map(&m0, g.w0, g.n, g.k, kMode == 2 ? 64 : 256));
  if (kMode == 2) GLMRT_RETURN_IF_ERROR(make_bytes_tensor_map(&m1, g.w1, g.n, g.k, 64));
  else m1 = m0;
  const size_t per = kMode == 0 ? 8 : 4;
  RowsArgs a{g.xs, g.ws0, g.ws1, g.out, g.out_scales, g.rows, g.n, g.k, g.xs_stride, g.out_stride,
             g.n % per == 0 && reinterpret_cast<uintptr_t>(g.out) % 16 == 0};
  static std::atomic<uint64_t> configured{0};
  GLMRT_RETURN_IF_ERROR(ensure_smem_limit(configured, fp8_rows_kernel<kMode>, kRowsSmem, "cudaFuncSetAttribute(fp8_rows_kernel)"));
  const int per_tile = kMode == 2 ? 128 : kRowsN;
  const long long tiles = static_cast<long long>((g.rows + 127) / 128) * ((g.n + per_tile - 1) / per_tile);
  launch_pdl(fp8_rows_kernel<kMode>, dim3(static_cast<unsigned>(std::min<long long>(tiles, sm_count))), dim3(kRowsThreads), kRowsSmem, s,
             a, mx, m0, m1);
  GLMRT_LAUNCH_CHECK("fp8_rows_kernel");
  return GLMRT_STATUS_OK;
}

// CTAs of a cluster that share a tile's K blocks: as many as fill the SMs once, at most eight and one per block.
int weight_splits(int n_tiles, int row_tiles, int blocks, int sm_count) {
  return std::max(1, std::min({8, blocks, sm_count / (n_tiles * row_tiles)}));
}

template <int kMode>
glmrt_status_t launch_mode(const Fp8Gemm& g, cudaStream_t s) {
  int dev = 0, sm_count = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, dev);
  const int n_tiles = (g.n + 127) / 128, blocks = (g.k + kFp8Block - 1) / kFp8Block;
  constexpr int kMostN = kMode == 2 ? 64 : 128;
  if (g.rows <= 128) {
    const int kn = g.rows <= 16 ? 16 : g.rows <= 32 ? 32 : g.rows <= 64 ? 64 : kMostN;
    const int splits = weight_splits(n_tiles, (g.rows + kn - 1) / kn, blocks, sm_count);
    if (kn == 16) return launch_weights<kMode, 16>(g, splits, s);
    if (kn == 32) return launch_weights<kMode, 32>(g, splits, s);
    if (kn == 64) return launch_weights<kMode, 64>(g, splits, s);
    if constexpr (kMode != 2) return launch_weights<kMode, 128>(g, splits, s);
  }
  return launch_rows<kMode>(g, sm_count, s);
}

}  // namespace

glmrt_status_t launch_fp8_gemm(const Fp8Gemm& g, int mode, cudaStream_t s) {
  return mode == 0 ? launch_mode<0>(g, s) : mode == 1 ? launch_mode<1>(g, s) : launch_mode<2>(g, s);
}

}  // namespace glmrt

using namespace glmrt;

extern "C" glmrt_status_t glmrt_b200_fp8_check(void* cuda_stream) {
  GLMRT_RETURN_IF_ERROR(require_cuda());
  uint32_t e = 0, zero = 0;
  cudaError_t err = cudaStreamSynchronize(static_cast<cudaStream_t>(cuda_stream));
  if (err == cudaSuccess) err = cudaMemcpyFromSymbol(&e, g_fp8_error, sizeof(e));
  if (err == cudaSuccess && e != 0) err = cudaMemcpyToSymbol(g_fp8_error, &zero, sizeof(zero));
  if (err != cudaSuccess) return fail_cuda(GLMRT_STATUS_COPY_FAILED, "fp8 check", err);
  return e == 0 ? ok() : fail(GLMRT_STATUS_INTERNAL_ERROR, "device reported: a bounded wait expired in an 8-bit product; its outputs are not valid");
}
