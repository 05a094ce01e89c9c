// Tensor-core products of the block-scaled 8-bit arithmetic (formats and definition: fp8.cu).
//
// tcgen05 kind::f8f6f4 multiplies a block of 128 columns at a time into tensor memory; the weight's
// scale is a general float32 per block, so the block sums cannot stay there: the epilogue warps read
// each one out, scale it and add it to float32 sums in their registers while the next block is
// multiplied into the other half of tensor memory.
//
//   rows on the MMA's lanes (fp8_rows_kernel)          many rows: tiles of 256 rows x 256 weight rows on CTA
//       pairs; a thread owns a row and 128 of its columns, so a block costs it one scale and 128 FMAs.
//   weights on the lanes (fp8_weights_kernel)          few rows: tiles of 128 weight rows x 16..128
//       rows, the K blocks of a tile split over a cluster of up to eight CTAs, whose sums meet in
//       shared memory.  Bound by the weight bytes, so what counts is that every SM streams.
//
// Measured (rows x n x k, in a chain of calls, the quantiser included): 8192 x 4096 x 6144 201 to 207 us = 2.0 PFLOP/s
// (float32 out 229), 8192 x 6144 x 2048 112 us; 1000 x 4096 x 6144 29 us, 256 rows 18.7, 64 rows 10.8, 16 rows 8.4; one row 6.8 us
// = 3.7 TB/s of weights from launch to launch, 5.6 between the first and the last copy.
//
// Each in two forms: the plain product, and gate / up with the SwiGLU and the next quantisation in the
// epilogue (both matrices in one tile, so that a thread meets gate and up of the same feature).
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "fp8.cuh"
#include "internal.h"
#include "tc_ptx.cuh"

namespace glmrt {
namespace {

using namespace tc;

__device__ uint32_t g_fp8_error;       // kErrWaitTimeout when a bounded wait ran out (glmrt_b200_operators_check)

// Brings a box into the L2.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
// Eight bf16 values as float32, zeros past the row's end (rows are multiples of 16 values).
__device__ __forceinline__ void quantise_load(const uint16_t* src, bool in, bool vec, float (&v)[8]) {
  uint16_t t[8] = {};
  if (in) {
    if (vec) {
      *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(src);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = src[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = bf16_bits_to_f32(t[i]);
}

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

// Keeps a CTA until the others of the cluster have read its shared memory: what they read went into what they stored,
// so nothing has to be made visible.  (A releasing arrival also waits for the stores to global memory: half a microsecond.)
__device__ __forceinline__ void cluster_leave() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// Two sums at once (fma.rn of each; for the few rows' kernel, 256 x 4096 x 6144 18.9 -> 17.8 us.  The many rows' has no
// register to spare for the pairs: 198 -> 252 us).
__device__ __forceinline__ void fma_pair(float& a0, float& a1, uint32_t v0, uint32_t v1, float s0, float s1) {
  asm("{\n\t.reg .b64 a, v, s;\n\t"
      "mov.b64 a, {%0, %1};\n\tmov.b64 v, {%2, %3};\n\tmov.b64 s, {%4, %5};\n\t"
      "fma.rn.f32x2 a, v, s, a;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "r"(v0), "r"(v1), "f"(s0), "f"(s1));
}

constexpr int kTileBytes = 128 * kFp8Block;            // 128 rows of one K block

// ---------------------------------------------------------------------------------------------------
// Many rows: tiles of 256 rows x 256 weight rows on CTA pairs (cta_group::2)
// ---------------------------------------------------------------------------------------------------
// Each CTA of a pair holds 128 of the rows and half of the weight rows, one M = 256 MMA of the leader
// fills a 128 x 256 block sum in each CTA's tensor memory.  A CTA alone would have to take in 48 KB per block's
// 512 cycles of multiplication, more than the 62 bytes a cycle that an SM gets from the L2; the pair needs 32 KB.
// A block takes 845 cycles (1.68 GHz under this load): an MMA 210 instead of 128, since its sums' way to tensor memory
// and back is shared with the epilogue's reading them out; a tile's end another 2200 that the two blocks ahead do not hide.
//
// Twelve warps: producer, issuer, two idle, eight epilogue warps (two per tensor-memory quadrant) that hold
// 128 sums a thread; registers move from the first four to them (3 x 128 threads x 168 = 128 x (40 + 2 x 232)).
constexpr int kPairStages = 5;
constexpr int kPairEpiWarps = 8;
constexpr int kPairThreads = 32 * (4 + kPairEpiWarps);
constexpr int kPairStageBytes = 2 * kTileBytes;                   // this CTA's rows and its half of the weight rows
constexpr int kPairN = 256;
constexpr int kBand = 8;                                          // row tiles of a band
constexpr int kParkWords = 36;                                    // a parked row: 32 words and four against bank conflicts
constexpr size_t kPairSmem = static_cast<size_t>(kPairStages) * kPairStageBytes + 1024 + 256 + 2 * 128 * 4 +
                             static_cast<size_t>(kPairEpiWarps) * 32 * kParkWords * 4;

struct RowsArgs {
  const float* xs;            // [blocks][xs_stride], whole tiles of 256 readable
  const float *ws0, *ws1;     // weight scales (gate / up: both)
  void* out;                  // product: [rows, n] bf16 or float32; SwiGLU: codes [rows, n]
  float* out_scales;          // SwiGLU: [ceil(n / 128)][out_stride]
  int rows, n, k, xs_stride, out_stride;
  int vector_out;             // whole 16-byte pieces: n and the output's address allow them
};

__device__ __forceinline__ void tc_mma_fp8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on the barrier at this place in both CTAs of the pair once every earlier product is done.
__device__ __forceinline__ void tc_commit_both(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}
// Arrival on the leader's barrier after reading tensor memory: the reads are complete (wait::ld) and ordered by the
// tcgen05 fence before it, no other memory has to become visible.  With .release.cluster the same arrival made the
// kernel wait for a memory barrier at every block (a third of its time).
__device__ __forceinline__ void mbar_arrive_remote(uint32_t bar_cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster_addr) : "memory");
}
__device__ __forceinline__ void tc_load32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]),
        "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
        "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}

// kMode 0: bf16 product, 1: float32 product, 2: SwiGLU of gate / up, quantised
template <int kMode>
__global__ void __launch_bounds__(kPairThreads, 1)
fp8_rows_kernel(RowsArgs a, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w0,
                const __grid_constant__ CUtensorMap map_w1) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + static_cast<size_t>(kPairStages) * kPairStageBytes);   // leader's count
  uint64_t* empty_bar = full_bar + kPairStages;      // one set per CTA
  uint64_t* acc_full = empty_bar + kPairStages;      // one pair per CTA
  uint64_t* acc_empty = acc_full + 2;                // leader's count
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  uint32_t* amax_x = reinterpret_cast<uint32_t*>(smem + static_cast<size_t>(kPairStages) * kPairStageBytes + 256);   // [2][128]
  uint32_t* park_all = amax_x + 256;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank();           // 0: leader
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int blocks = (a.k + kFp8Block - 1) / kFp8Block;
  const int per_tile = kMode == 2 ? 128 : kPairN;                 // output columns of a tile
  const int n_tiles = (a.n + per_tile - 1) / per_tile, m_tiles = (a.rows + 255) / 256;
  const int tiles = n_tiles * m_tiles;

  if (threadIdx.x == 32) {
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w0);
    if (kMode == 2) prefetch_tensormap(&map_w1);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * kPairEpiWarps);
    }
    *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  cluster_sync_all();           // barriers of both CTAs initialised, tensor memory of both allocated
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();      // after the wait: a successor may then rely on everything before this kernel

  // Tiles in bands of eight row tiles, column by column inside a band, so that the tiles in flight (74 pairs) form
  // a block of about 8 x 9 whose rows and weights stay in the L2 while they are read.
  auto tile_at = [&](int tile, int& m, int& nt) {
    const int band = tile / (kBand * n_tiles), in = tile - band * kBand * n_tiles;
    const int high = min(kBand, m_tiles - band * kBand);
    nt = in / high;
    m = band * kBand + in - nt * high;
  };
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
      const uint64_t pol = policy_evict_last();
      int stage = 0;
      uint32_t phase = 0;
      bool alive = true;
      for (int tile = pair; tile < tiles && alive; tile += pairs) {
        int mt, nt;
        tile_at(tile, mt, nt);
        const int m0 = mt * 256 + 128 * static_cast<int>(rank), n0 = nt * per_tile;
        for (int b = 0; b < blocks; ++b) {
          if (!mbar_wait_hot(&empty_bar[stage], phase ^ 1u, abort_flag)) { alive = false; break; }
          if (elect_one()) {
            const uint32_t s_a = smem_u32(smem + static_cast<size_t>(stage) * kPairStageBytes), s_b = s_a + kTileBytes;
            const uint32_t full = cluster_addr(smem_u32(&full_bar[stage]), 0);
            if (rank == 0) mbar_expect_tx(&full_bar[stage], 2 * kPairStageBytes);
            tma_load_2d_pair(s_a, &map_x, full, b * kFp8Block, m0, pol);
            if (kMode == 2) {     // this CTA's 64 features: their gate rows, then their up rows
              tma_load_2d_pair(s_b, &map_w0, full, b * kFp8Block, n0 + 64 * static_cast<int>(rank), pol);
              tma_load_2d_pair(s_b + kTileBytes / 2, &map_w1, full, b * kFp8Block, n0 + 64 * static_cast<int>(rank), pol);
            } else {
              tma_load_2d_pair(s_b, &map_w0, full, b * kFp8Block, n0 + 128 * static_cast<int>(rank), pol);
            }
          }
          __syncwarp();
          if (++stage == kPairStages) { stage = 0; phase ^= 1u; }
        }
      }
    } else if (warp == 1 && rank == 0) {
      int stage = 0, abuf = 0;
      uint32_t phase = 0, aphase = 0;
      bool alive = true;
      const uint32_t idesc = (1u << 4) | ((static_cast<uint32_t>(kPairN) >> 3) << 17) | ((256u >> 4) << 24);
      for (int tile = pair; tile < tiles && alive; tile += pairs)
        for (int b = 0; b < blocks; ++b) {
          // (the copies are early, the sums' buffer is what the next product waits for: its wait comes last)
          const bool ready = mbar_wait_lane(&full_bar[stage], phase, abort_flag) && mbar_wait_lane(&acc_empty[abuf], aphase ^ 1u, abort_flag);
          tc_fence_after();
          if (elect_one() && ready) {
            const uint32_t s_a = smem_u32(smem + static_cast<size_t>(stage) * kPairStageBytes), s_b = s_a + kTileBytes;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc_mma_fp8_pair(tmem_base + abuf * kPairN, desc_sw128(s_a + kk * 32), desc_sw128(s_b + kk * 32), idesc, kk != 0 ? 1u : 0u);
            tc_commit_both(&acc_full[abuf]);
            tc_commit_both(&empty_bar[stage]);
          }
          // The lanes' answers meet only now: before the products the vote would cost 3 % of a large product's time
          // (8192 x 6144 x 2048: 114.2 us, here 112.5).
          if (!__all_sync(0xffffffffu, ready)) { alive = false; break; }
          if (++stage == kPairStages) { stage = 0; phase ^= 1u; }
          abuf ^= 1;
          if (abuf == 0) aphase ^= 1u;
        }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int quad = warp & 3, part = (warp - 4) >> 2;       // tensor-memory lanes, half of the tile's columns
    const int lane_row = quad * 32 + lane;
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + part * 128;
    const uint32_t lead_acc_empty = cluster_addr(smem_u32(acc_empty), 0);
    uint32_t* park = park_all + (warp - 4) * 32 * kParkWords;
    int abuf = 0;
    uint32_t aphase = 0;
    // A warp whose wait ran out keeps step with the others (they meet at barriers), computing nothing valid.
    for (int tile = pair; tile < tiles; tile += pairs) {
      int mt, nt;
      tile_at(tile, mt, nt);
      const int row0 = mt * 256 + 128 * static_cast<int>(rank) + quad * 32, row = row0 + lane;
      const int n0 = nt * per_tile;
      // the product's halves are two weight blocks; gate and up share the block number of their features
      const int wb = kMode == 2 ? nt : min(nt * 2 + part, (a.n - 1) / kFp8Block);
      const float* xs = a.xs + row;
      const float* ws0 = a.ws0 + static_cast<size_t>(wb) * blocks;
      const float* ws1 = kMode == 2 ? a.ws1 + static_cast<size_t>(wb) * blocks : ws0;
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
      float sx = __ldg(xs), w0 = __ldg(ws0), w1 = __ldg(ws1);
      for (int b = 0; b < blocks; ++b) {
        const float s0 = sx * w0, s1 = sx * w1;
        if (b + 1 < blocks) {       // the next block's scales come from the L2 under this block
          sx = __ldg(xs + static_cast<size_t>(b + 1) * a.xs_stride);
          w0 = __ldg(ws0 + b + 1);
          if (kMode == 2) w1 = __ldg(ws1 + b + 1);
          else w1 = w0;
        }
        mbar_wait_lane(&acc_full[abuf], aphase, abort_flag);
        __syncwarp();
        tc_fence_after();
        const uint32_t t = t_lane + abuf * kPairN;
        // 64 columns in flight at a time; the buffer is free again before the last half is added
        uint32_t v[2][32];
        tc_load32(t, v[0]);
        tc_load32(t + 32, v[1]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          tc_wait_ld();
          if (half == 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(lead_acc_empty + abuf * 8);
          }
          const float s = kMode == 2 && half == 1 ? s1 : s0;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              acc[half * 64 + c * 32 + i] = fmaf(__uint_as_float(v[c][i]), s, acc[half * 64 + c * 32 + i]);
            if (half == 0) tc_load32(t + 64 + c * 32, v[c]);
          }
        }
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
        amax_x[part * 128 + lane_row] = amax;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kPairEpiWarps) : "memory");
        amax = max(amax, amax_x[(part ^ 1) * 128 + lane_row]);
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kPairEpiWarps) : "memory");   // read before the next tile writes
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
      } else {
        // Through shared memory, 32 words of each of the warp's rows at a time, so that a row leaves as 128
        // consecutive bytes (a word is two bf16 or one float32), four rows an instruction.
        constexpr int kPer = kMode == 0 ? 2 : 1;
#pragma unroll
        for (int pass = 0; pass < 4 / kPer; ++pass) {
          const int c0 = n0 + 128 * part + pass * 32 * kPer;
          auto word = [&](int i) {
            return kMode == 0 ? pack_bf16x2(acc[pass * 32 * kPer + i * kPer], acc[pass * 32 * kPer + i * kPer + kPer - 1])
                              : __float_as_uint(acc[pass * 32 * kPer + i]);
          };
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(park + lane * kParkWords + i) = make_uint4(word(i), word(i + 1), word(i + 2), word(i + 3));
          __syncwarp();
          using Out = typename std::conditional<kMode == 0, uint16_t, float>::type;
          Out* out = static_cast<Out*>(a.out) + static_cast<size_t>(row0) * a.n + c0;
          if (a.vector_out) {
            const int c = (lane & 7) * 4 * kPer;
            if (c0 + c < a.n) {
#pragma unroll
              for (int r = lane >> 3; r < 32; r += 4)
                if (row0 + r < a.rows)
                  *reinterpret_cast<uint4*>(out + static_cast<size_t>(r) * a.n + c) =
                      *reinterpret_cast<const uint4*>(park + r * kParkWords + (lane & 7) * 4);
            }
          } else {
            const Out* src = reinterpret_cast<const Out*>(park);
            for (int r = 0; r < 32 && row0 + r < a.rows; ++r)
#pragma unroll
              for (int c = lane; c < 32 * kPer; c += 32)
                if (c0 + c < a.n) out[static_cast<size_t>(r) * a.n + c] = src[r * kParkWords * kPer + c];
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
  cluster_sync_all();           // neither CTA frees tensor memory the other may still be written through
  if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
}

// ---------------------------------------------------------------------------------------------------
// Few rows
// ---------------------------------------------------------------------------------------------------
struct WeightsArgs {
  const float* xs;            // [blocks][xs_stride] (quantised in the kernel: unused)
  const uint16_t* x;          // bf16 rows x_stride apart, quantised in the kernel; else unused
  size_t x_stride;
  int x_vector;               // the rows start on 16-byte boundaries
  const float *ws0, *ws1;
  void* out;
  float* out_scales;
  int rows, n, k, xs_stride, out_stride;
};

// kOwnX: the rows are bf16 and every CTA quantises the blocks it needs itself (a few rows: one launch less than
// quantising them first, and no workspace); their codes lie beside the ring, kXBlocks blocks at a time.
template <int kMode, int kN, bool kOwnX>
struct WCfg {
  static constexpr int kMats = kMode == 2 ? 2 : 1;
  static constexpr int kStageBytes = kMats * kTileBytes + (kOwnX ? 0 : kN * kFp8Block);
  static constexpr int kXBlocks = kMode == 2 ? 6 : 8;
  static constexpr int kXBytes = kOwnX ? kXBlocks * kN * kFp8Block : 0;
  static constexpr int kAccCols = kMats * kN;                       // of one block
  // Two CTAs on an SM where the sums leave the registers for it: twice as many chains of copy, product and
  // read-out side by side, and twice as many splits of a tile.
  static constexpr int kPerSm = kAccCols <= 64 ? 2 : 1;
  static constexpr int kRingBytes = (kPerSm == 2 ? (kOwnX ? 111616 : 104448) : 184320) - kXBytes;
  static constexpr int kStages = kRingBytes / kStageBytes < 8 ? kRingBytes / kStageBytes : 8;
  static constexpr int kScaleBlocks = kOwnX ? kXBlocks : 16;        // blocks whose scales are kept in shared memory
  static constexpr int kTmemCols = 2 * kAccCols < 32 ? 32 : 2 * kAccCols;
  static constexpr int kParts = kAccCols > 64 ? 2 : 1;              // epilogue warps per tensor-memory quadrant, by columns
  static constexpr int kEpiWarps = 4 * kParts;
  static constexpr int kCols = kN / kParts;                         // of each matrix, per thread
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr size_t kSmem = static_cast<size_t>(kStages) * kStageBytes + kXBytes + 1024 + 512 + kScaleBlocks * kN * kMats * 4;
  static_assert(static_cast<size_t>(kStages) * kStageBytes >= static_cast<size_t>(kMats) * kN * 128 * 4, "partial sums reuse the ring");
};

// grid (weight tiles, splits, row tiles), cluster (1, splits, 1).
// One row, 4096 x 6144, in ns after its rows are there: first block 800, last block 5200 (12 blocks a CTA), sums
// joined 5800, stored 6100.  More block sums in tensor memory than two (no wait for the read-out), or all of a CTA's
// weights asked into the L2 ahead instead of a ring's, gained nothing.
template <int kMode, int kN, bool kOwnX>
__global__ void __launch_bounds__(WCfg<kMode, kN, kOwnX>::kThreads, WCfg<kMode, kN, kOwnX>::kPerSm)
fp8_weights_kernel(WeightsArgs a, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w0,
                   const __grid_constant__ CUtensorMap map_w1) {
  using C = WCfg<kMode, kN, kOwnX>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* x_codes = smem + static_cast<size_t>(C::kStages) * C::kStageBytes;      // kOwnX: [kXBlocks] tiles of kN rows
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(x_codes + C::kXBytes);
  uint64_t* empty_bar = full_bar + C::kStages;
  uint64_t* acc_full = empty_bar + C::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* x_full = acc_empty + 2;                                                 // kOwnX: a group of blocks is quantised
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(x_full + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  // scales of the next blocks, row's times weight's (a power of two: exact): [kMats][kScaleBlocks][kN]
  float* scale_all = reinterpret_cast<float*>(x_codes + C::kXBytes + 512);

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
      mbar_init(&acc_empty[b], C::kEpiWarps);
    }
    mbar_init(x_full, C::kEpiWarps);
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
    // The previous kernel of this call let this one start only after everything before it had finished, and wrote no
    // weights: the first stages' weights are asked for before its rows are waited for.  Where this kernel is the
    // call's first, they are only brought into the L2 until then.
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
      for (int i = 0; i < ahead; ++i) {
        if constexpr (kOwnX) {
          tma_prefetch_2d(&map_w0, (b0 + i) * kFp8Block, w0);
          if (kMode == 2) tma_prefetch_2d(&map_w1, (b0 + i) * kFp8Block, w0);
        } else {
          load_w(i, b0 + i);
        }
      }
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();
    if (elect_one())
      for (int i = 0; i < ahead; ++i) {
        if constexpr (kOwnX) load_w(i, b0 + i);
        else load_x(i, b0 + i);
      }
    __syncwarp();
    int stage = 0;
    uint32_t phase = 0;
    for (int b = b0 + ahead; b < b1; ++b) {
      if (!mbar_wait_hot(&empty_bar[stage], phase, abort_flag)) break;
      if (elect_one()) {
        load_w(stage, b);
        if constexpr (!kOwnX) load_x(stage, b);
      }
      __syncwarp();
      if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
    }
  } else if (warp == 1) {
    pdl_wait();
    int stage = 0, abuf = 0;
    uint32_t phase = 0, aphase = 0;
    const uint32_t idesc = idesc_fp8(kN);
    uint32_t xphase = 0;
    for (int b = b0; b < b1; ++b) {
      if (kOwnX && (b - b0) % C::kXBlocks == 0) {
        if (!mbar_wait_hot(x_full, xphase, abort_flag)) break;
        xphase ^= 1u;
      }
      const bool ready = mbar_wait_lane(&acc_empty[abuf], aphase ^ 1u, abort_flag) && mbar_wait_lane(&full_bar[stage], phase, abort_flag);
      tc_fence_after();
      if (elect_one() && ready) {
        const uint32_t s_a = smem_u32(smem + static_cast<size_t>(stage) * C::kStageBytes), s_x = kOwnX ? smem_u32(x_codes) + (b - b0) % C::kXBlocks * kN * kFp8Block : s_a + C::kMats * kTileBytes;
#pragma unroll
        for (int mat = 0; mat < C::kMats; ++mat)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc_mma_fp8(tmem_base + abuf * C::kAccCols + mat * kN, desc_sw128(s_a + mat * kTileBytes + kk * 32),
                       desc_sw128(s_x + kk * 32), idesc, kk != 0 ? 1u : 0u);
        tc_commit(&empty_bar[stage]);
        tc_commit(&acc_full[abuf]);
      }
      if (!__all_sync(0xffffffffu, ready)) break;      // (after the products, as in the kernel above)
      if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
      abuf ^= 1;
      if (abuf == 0) aphase ^= 1u;
    }
  }
  const int quad = warp & 3, lane_row = quad * 32 + lane;           // epilogue warps: weight row of the tile
  const int part_col = ((warp - 2) >> 2) * C::kCols;                // first column of this warp's share
  float acc[C::kMats][C::kCols];
  if (warp >= 2) {
    pdl_wait();
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + part_col;
    const size_t wb = static_cast<size_t>(blockIdx.x) * blocks;
#pragma unroll
    for (int mat = 0; mat < C::kMats; ++mat)
#pragma unroll
      for (int j = 0; j < C::kCols; ++j) acc[mat][j] = 0.0f;
    int abuf = 0;
    uint32_t aphase = 0;
    const int tid = threadIdx.x - 64;
    for (int b = b0; b < b1; ++b) {
      const int at = (b - b0) % C::kScaleBlocks;
      if (at == 0) {              // the scales of the next blocks (rows padded to whole tiles)
        const int count = min(C::kScaleBlocks, b1 - b);
        asm volatile("bar.sync 1, %0;" ::"n"(32 * C::kEpiWarps) : "memory");
        if constexpr (kOwnX) {
          // The products of the blocks before have all been read out, so their codes may go.  Half a warp per (row,
          // block), eight values a lane, stored where the 128-byte swizzle puts them.
          const int sub = tid % 16, rows = min(kN, a.rows - m0);
          for (int i = tid / 16; i < count * rows; i += 2 * C::kEpiWarps) {
            const int row = i / count, bb = i - row * count, c = (b + bb) * kFp8Block + sub * 8;
            float v[8];
            quantise_load(a.x + static_cast<size_t>(m0 + row) * a.x_stride + c, c < a.k, a.x_vector != 0, v);
            uint32_t amax = 0u;
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(v[e]) & 0x7fffffffu);
            const uint32_t half = 0xffffu << (threadIdx.x & 16);       // the lanes of this row and block
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(half, amax, o));
            float inv;
            const float scale = fp8_block_scale(amax, &inv);
            *reinterpret_cast<uint2*>(x_codes + bb * kN * kFp8Block + row * kFp8Block + (((sub >> 1) ^ (row & 7)) << 4) + (sub & 1) * 8) =
                make_uint2(fp8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv), fp8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
            if (sub == 0) {
              scale_all[bb * kN + row] = scale * __ldg(a.ws0 + wb + b + bb);
              if (kMode == 2) scale_all[(C::kScaleBlocks + bb) * kN + row] = scale * __ldg(a.ws1 + wb + b + bb);
            }
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(x_full);
        } else {
          for (int i = tid; i < count * (kN / 4); i += 32 * C::kEpiWarps) {
            const int bb = i / (kN / 4);
            const float4 sx = *reinterpret_cast<const float4*>(a.xs + static_cast<size_t>(b + bb) * a.xs_stride + m0 + (i % (kN / 4)) * 4);
#pragma unroll
            for (int mat = 0; mat < C::kMats; ++mat) {
              const float sw = __ldg((mat == 0 ? a.ws0 : a.ws1) + wb + b + bb);
              reinterpret_cast<float4*>(scale_all)[mat * C::kScaleBlocks * (kN / 4) + i] = make_float4(sx.x * sw, sx.y * sw, sx.z * sw, sx.w * sw);
            }
          }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * C::kEpiWarps) : "memory");
      }
      const float* scales = scale_all + at * kN + part_col;
      mbar_wait_lane(&acc_full[abuf], aphase, abort_flag);     // on a time-out it keeps step, computing nothing valid
      __syncwarp();
      tc_fence_after();
      // Chunks of all matrices' columns, the next one's on their way while one is added.
      constexpr int kChunk = C::kCols >= 32 ? 32 : 16, kChunks = C::kMats * C::kCols / kChunk;
      uint32_t v[2][kChunk];
      auto load = [&](int c, uint32_t (&dst)[kChunk]) {
        const uint32_t at_col = t_lane + abuf * C::kAccCols + c * kChunk / C::kCols * kN + c * kChunk % C::kCols;
        if constexpr (kChunk == 32) tc_load32(at_col, dst);
        else tc_load16(at_col, dst);
      };
      load(0, v[0]);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        tc_wait_ld();
        if (c + 1 < kChunks) load(c + 1, v[(c + 1) & 1]);
        const int mat = c * kChunk / C::kCols, col = c * kChunk % C::kCols;
#pragma unroll
        for (int i = 0; i < kChunk; i += 4) {
          const float4 q = *reinterpret_cast<const float4*>(scales + mat * C::kScaleBlocks * kN + col + i);
          fma_pair(acc[mat][col + i], acc[mat][col + i + 1], v[c & 1][i], v[c & 1][i + 1], q.x, q.y);
          fma_pair(acc[mat][col + i + 2], acc[mat][col + i + 3], v[c & 1][i + 2], v[c & 1][i + 3], q.z, q.w);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[abuf]);
      abuf ^= 1;
      if (abuf == 0) aphase ^= 1u;
    }
  }

  // ---- the splits' sums meet: [matrix][row of x][weight row] in each CTA's ring.  An epilogue warp has seen the last
  // product done, so nobody reads the ring any more and all its copies have landed. ----
  tc_fence_before();
  float* part = reinterpret_cast<float*>(smem);
  if (warp >= 2)
#pragma unroll
    for (int mat = 0; mat < C::kMats; ++mat)
#pragma unroll
      for (int j = 0; j < C::kCols; ++j) part[(mat * kN + part_col + j) * 128 + lane_row] = acc[mat][j];
  if (splits > 1) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, C::kTmemCols);
  if (*abort_flag != 0u) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);   // let copies in flight land
    if (threadIdx.x == 0) atomicOr(&g_fp8_error, static_cast<uint32_t>(kErrWaitTimeout));
  }
  // This CTA finishes rows j0 .. j1 of the tile, one warp a row and four features a lane, the splits added in order.
  // A load from another CTA's shared memory takes most of a microsecond, so a lane has all splits' in flight.
  const int valid = min(kN, a.rows - m0);
  const int j0 = valid * split / splits, j1 = valid * (split + 1) / splits;
  if (warp >= 2) {
    const uint32_t part_at = smem_u32(part) + lane * 16;
    const int feature = w0 + lane * 4;
    constexpr int kBatch = kMode == 2 ? 1 : 2;
    for (int jb = j0 + (warp - 2) * kBatch; jb < j1; jb += C::kEpiWarps * kBatch) {
      float v[C::kMats * kBatch][8][4];
#pragma unroll
      for (int q = 0; q < C::kMats * kBatch; ++q) {
        const int j = kMode == 2 ? q * kN + jb : jb + q;       // gate and up of one row, or two rows
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          v[q][r][0] = v[q][r][1] = v[q][r][2] = v[q][r][3] = 0.0f;
          if (r < splits && (kMode == 2 || j < j1))
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v[q][r][0]), "=f"(v[q][r][1]), "=f"(v[q][r][2]), "=f"(v[q][r][3])
                         : "r"(cluster_addr(part_at + j * 512, r))
                         : "memory");
        }
      }
      float y[C::kMats * kBatch][4];
#pragma unroll
      for (int q = 0; q < C::kMats * kBatch; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[q][i] = v[q][0][i];
#pragma unroll
          for (int r = 1; r < 8; ++r) y[q][i] += v[q][r][i];
        }
      if constexpr (kMode == 2) {
        // SwiGLU, and the block's (128 features of one row) scale
        uint32_t amax = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[0][i] = fp8_swiglu(y[0][i], y[1][i]);
          amax = max(amax, __float_as_uint(y[0][i]) & 0x7fffffffu);
        }
        float inv;
        const float scale = fp8_block_scale(__reduce_max_sync(0xffffffffu, amax), &inv);
        const size_t row = static_cast<size_t>(m0 + jb);
        if (feature < a.n)                                      // n % 16 == 0
          *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.out) + row * a.n + feature) =
              fp8_pack4(y[0][0] * inv, y[0][1] * inv, y[0][2] * inv, y[0][3] * inv);
        if (lane == 0) a.out_scales[static_cast<size_t>(blockIdx.x) * a.out_stride + row] = scale;
      } else {
        using Out = typename std::conditional<kMode == 0, uint16_t, float>::type;
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
          if (jb + q >= j1) break;
          Out* out = static_cast<Out*>(a.out) + static_cast<size_t>(m0 + jb + q) * a.n + feature;
          if (feature + 3 < a.n && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(Out)) == 0) {
            if constexpr (kMode == 0) *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(y[q][0], y[q][1]), pack_bf16x2(y[q][2], y[q][3]));
            else *reinterpret_cast<float4*>(out) = make_float4(y[q][0], y[q][1], y[q][2], y[q][3]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (feature + i < a.n) fp8_store(out + i, y[q][i]);
          }
        }
      }
    }
  }
  if (splits > 1) cluster_leave();          // nobody leaves while its sums may still be read
}

constexpr int kMaxDevices = 64;

// Clusters of `splits` CTAs that run at once on the current device (they must fit into one GPC each, so this is
// less than the SMs divided by the size); asked once per device.
template <int kMode, int kN, bool kOwnX>
int active_clusters(int dev, int splits) {
  using C = WCfg<kMode, kN, kOwnX>;
  static std::atomic<int> known[kMaxDevices][9];
  if (dev < 0 || dev >= kMaxDevices) return 0;
  int n = known[dev][splits].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(1, static_cast<unsigned>(splits), 1);
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1; attr[0].val.clusterDim.y = static_cast<unsigned>(splits); attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, fp8_weights_kernel<kMode, kN, kOwnX>, &cfg) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    known[dev][splits].store(n, std::memory_order_relaxed);
  }
  return n;
}

// CTAs of a cluster that share a tile's K blocks: the number with the shortest estimated time.  A wave of CTAs
// costs about 3 us beside its blocks (set-up, first copies, joining), a block 0.42 us and 0.0015 us per column of
// the sum (measured at 16 to 256 rows and 2048 to 6144 columns of K).  The driver's count is that of one CTA an SM.
// With rows quantised here a second one beside it helps, since each CTA then has fewer blocks of them (1 row, n x k:
// 4096 x 6144 4 splits 8.3 us, 6 splits 6.8; 12288 x 4096 1 split 15.9, 2 splits 10.6); otherwise it does not (16 rows,
// 4096 x 6144: 4 splits 8.4, 6 splits 8.7; 64 rows 10.9 / 11.9).
template <int kMode, int kN, bool kOwnX>
int weight_splits(int tiles, int blocks, float* estimate_us) {
  int best = 1, dev = 0;
  cudaGetDevice(&dev);
  float best_us = 0.0f;
  for (int s = 1; s <= 8 && s <= blocks; ++s) {
    const int active = active_clusters<kMode, kN, kOwnX>(dev, s) * (kOwnX ? WCfg<kMode, kN, kOwnX>::kPerSm : 1);
    if (active <= 0) continue;
    const float us = static_cast<float>((tiles + active - 1) / active) *
                     (3.0f + (s > 1 ? 0.7f : 0.0f) + static_cast<float>((blocks + s - 1) / s) * (0.42f + 0.0015f * WCfg<kMode, kN, kOwnX>::kAccCols));
    if (best_us == 0.0f || us < best_us) { best = s; best_us = us; }
  }
  *estimate_us = best_us;
  return best;
}

template <int kMode, int kN, bool kOwnX = false>
glmrt_status_t launch_weights(const Fp8Gemm& g, cudaStream_t s) {
  using C = WCfg<kMode, kN, kOwnX>;
  static std::atomic<uint64_t> configured{0};
  GLMRT_RETURN_IF_ERROR(ensure_smem_limit(configured, fp8_weights_kernel<kMode, kN, kOwnX>, C::kSmem, "cudaFuncSetAttribute(fp8_weights_kernel)"));
  float us = 0.0f;
  const int splits = weight_splits<kMode, kN, kOwnX>((g.n + 127) / 128 * ((g.rows + kN - 1) / kN), (g.k + kFp8Block - 1) / kFp8Block, &us);
  CUtensorMap mx, m0, m1;
  GLMRT_RETURN_IF_ERROR(make_bytes_tensor_map(&m0, g.w0, g.n, g.k, 128));
  if (kMode == 2) GLMRT_RETURN_IF_ERROR(make_bytes_tensor_map(&m1, g.w1, g.n, g.k, 128));
  else m1 = m0;
  if (kOwnX) mx = m0;
  else GLMRT_RETURN_IF_ERROR(make_bytes_tensor_map(&mx, g.x, g.rows, g.k, kN));
  WeightsArgs a{g.xs, g.x_bf16, g.x_stride, g.x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(g.x_bf16) % 16 == 0, g.ws0, g.ws1, g.out, g.out_scales, g.rows, g.n, g.k, g.xs_stride, g.out_stride};
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
  cudaError_t err = cudaLaunchKernelEx(&cfg, fp8_weights_kernel<kMode, kN, kOwnX>, a, mx, m0, m1);
  if (err != cudaSuccess) return fail_cuda(GLMRT_STATUS_COPY_FAILED, "fp8_weights_kernel", err);
  GLMRT_LAUNCH_CHECK("fp8_weights_kernel");
  return GLMRT_STATUS_OK;
}

template <int kMode>
glmrt_status_t launch_rows(const Fp8Gemm& g, int sm_count, cudaStream_t s) {
  CUtensorMap mx, m0, m1;
  GLMRT_RETURN_IF_ERROR(make_bytes_tensor_map(&mx, g.x, g.rows, g.k, 128));
  GLMRT_RETURN_IF_ERROR(make_bytes_tensor_map(&m0, g.w0, g.n, g.k, kMode == 2 ? 64 : 128));
  if (kMode == 2) GLMRT_RETURN_IF_ERROR(make_bytes_tensor_map(&m1, g.w1, g.n, g.k, 64));
  else m1 = m0;
  RowsArgs a{g.xs, g.ws0, g.ws1, g.out, g.out_scales, g.rows, g.n, g.k, g.xs_stride, g.out_stride,
             g.n % (kMode == 0 ? 8 : 4) == 0 && reinterpret_cast<uintptr_t>(g.out) % 16 == 0};
  static std::atomic<uint64_t> configured{0};
  GLMRT_RETURN_IF_ERROR(ensure_smem_limit(configured, fp8_rows_kernel<kMode>, kPairSmem, "cudaFuncSetAttribute(fp8_rows_kernel)"));
  const int per_tile = kMode == 2 ? 128 : kPairN;
  const long long tiles = static_cast<long long>((g.rows + 255) / 256) * ((g.n + per_tile - 1) / per_tile);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min<long long>(tiles, sm_count / 2)));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t err = cudaLaunchKernelEx(&cfg, fp8_rows_kernel<kMode>, a, mx, m0, m1);
  if (err != cudaSuccess) return fail_cuda(GLMRT_STATUS_COPY_FAILED, "fp8_rows_kernel", err);
  GLMRT_LAUNCH_CHECK("fp8_rows_kernel");
  return GLMRT_STATUS_OK;
}

// Tiles of 16, 32 and 64 rows for batches that small.  Above, the larger of the weight-row tiles or the row tiles,
// by their estimates: a wave of row tiles costs about 4 us and 0.48 us a block, whatever part of its 256 rows is
// filled (measured, row tiles against weight-row tiles: 256 rows, n = 6144, k = 2048 12.3 / 13.8 us; n = 4096, k = 6144
// 24 / 18; n = 1500, k = 2000 15 / 9; 600 rows, n = 4096, k = 6144 26 / 49).
constexpr int kWeightsMostRows = 1024;

template <int kMode>
glmrt_status_t launch_mode(const Fp8Gemm& g, cudaStream_t s) {
  constexpr int kMostN = kMode == 2 ? 64 : 128;
  if (g.x_bf16 != nullptr) return launch_weights<kMode, 16, true>(g, s);      // at most kFp8OwnRows rows
  if (g.rows <= 16) return launch_weights<kMode, 16>(g, s);
  if (g.rows <= 32) return launch_weights<kMode, 32>(g, s);
  if (g.rows <= 64) return launch_weights<kMode, 64>(g, s);
  int dev = 0, sm_count = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, dev);
  if (g.rows <= kWeightsMostRows) {
    using C = WCfg<kMode, kMostN, false>;
    static std::atomic<uint64_t> configured{0};
    GLMRT_RETURN_IF_ERROR(ensure_smem_limit(configured, fp8_weights_kernel<kMode, kMostN, false>, C::kSmem, "cudaFuncSetAttribute(fp8_weights_kernel)"));
    const int blocks = (g.k + kFp8Block - 1) / kFp8Block, per_tile = kMode == 2 ? 128 : kPairN;
    const int tiles = (g.n + 127) / 128 * ((g.rows + kMostN - 1) / kMostN);
    const int row_tiles = (g.n + per_tile - 1) / per_tile * ((g.rows + 255) / 256), pairs = sm_count / 2;
    float us = 0.0f;
    weight_splits<kMode, kMostN, false>(tiles, blocks, &us);
    if (us < static_cast<float>((row_tiles + pairs - 1) / pairs) * (4.0f + 0.48f * static_cast<float>(blocks)))
      return launch_weights<kMode, kMostN>(g, s);
  }
  return launch_rows<kMode>(g, sm_count, s);
}

}  // namespace

glmrt_status_t launch_fp8_gemm(const Fp8Gemm& g, int mode, cudaStream_t s) {
  return mode == 0 ? launch_mode<0>(g, s) : mode == 1 ? launch_mode<1>(g, s) : launch_mode<2>(g, s);
}
glmrt_status_t fp8_take_error(uint32_t* out) { return take_error_word(g_fp8_error, out); }

}  // namespace glmrt

using namespace glmrt;

extern "C" glmrt_status_t glmrt_b200_operators_check(void* cuda_stream) {
  GLMRT_RETURN_IF_ERROR(require_cuda());
  uint32_t fp8 = 0, norm = 0;
  cudaError_t err = cudaStreamSynchronize(static_cast<cudaStream_t>(cuda_stream));
  if (err != cudaSuccess) return fail_cuda(GLMRT_STATUS_COPY_FAILED, "operators check", err);
  GLMRT_RETURN_IF_ERROR(fp8_take_error(&fp8));
  GLMRT_RETURN_IF_ERROR(norm_take_error(&norm));
  if ((fp8 | norm) == 0) return ok();
  return fail(GLMRT_STATUS_INTERNAL_ERROR, std::string("device reported: a bounded wait expired in ") + (fp8 ? "an 8-bit product" : "a block norm") +
                                               "; its outputs are not valid");
}
