// A whole sparse layer for a few tokens (at most kFewMaxRows rows): router, experts on bf16
// activations (W4A16, the arithmetic of the reference's decode kernels: native/cuda/kernels/
// b12x_direct.cu:171-201,989-1541), weighted combine, and the residual and shared rows added on top.
//
//   act[r]  = weight[r] * silu(gate x) * (up x)          r = (token, slot), float32
//   out[t]  = residual[t] + (shared[t] + sum over slots down act[t, slot])
//
// with W = E2M1 code * E4M3 block scale * scale_2.  Between the bf16 rows and the bf16 result only the SwiGLU rows are
// rounded to fewer bits than float32, and rows of very wide range (both below); the verification form rounds neither.
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "tc_ptx.cuh"

namespace glmrt {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ------------------------------------------------------------------------------------------------
// One cooperative kernel, one CTA per SM, three grid-wide barriers:
//
//   logits     every warp: one expert x one share of the hidden columns, float32 weights       | barrier
//   selection  every CTA for itself: sigmoid, top-k, the list of (expert, one or two tokens) entries
//   gate / up  the entries' rows split evenly over the CTAs                                    | barrier
//   down       the same; one float32 row per route                                             | barrier
//   combine    residual + (shared + sum over the slots, in slot order)
//
// What bounds it is the experts' weights (9/16 byte each, read once); everything else is arranged so
// that they never stop arriving.  Measured at 6144 / 2048, 256 experts, top-8, back to back: 1 row 48 us (170 MB; 9 us
// until the routes are known, 19 us gate / up, 2 us barrier, 11 us down, 5 us barrier and combine), 4 rows 130, 8 rows
// 235 to 262, 16 rows 429 to 462 us (2.2 GB: 4.7 to 5.1 TB/s, by then bound by issue slots, 295 instructions a slot).  Each lane copies its own pieces of the weights into shared memory
// (cp.async), kRing - 1 slots ahead, and only itself reads them back, so the stream needs no barrier
// between warps; it runs on from the gate / up rows into the down rows while the CTA waits at the
// barrier between them.
//
// A piece is 16 weight rows x 128 columns of one warp: 16 B of codes of each of two rows per lane (32
// columns) and the scales of both.  A slot is two pieces at the same columns: the same rows of gate and up,
// or 32 rows of down.  E2M1 codes become fp16 pairs (one instruction for two) and the tensor cores multiply
// them (m16n8k16, float32 sums).  Which columns a lane holds does not matter as long as both operands agree,
// so lane t of a row's four takes columns 32t .. 32t+31, two scale blocks.  A product's four lanes thus lie in
// four different blocks; to keep the blocks apart an entry has at most two tokens and a token four of the
// eight columns, column t' holding the token's values of lane t' and zeros elsewhere.  So a sum of four products
// is one block's, and the E4M3 scale is multiplied to it in float32: 16 FMAs a slot, where scaling the weights
// themselves takes 64 fp16 multiplications on the pipe that the products run on (measured: 18.5 cycles a product
// with them, 10.5 without; the conversions take 12 on another pipe).
//
// The rows as fp16: times a power of two per token that brings the largest magnitude to 2^14, which is
// exact for everything within 2^28 of it and off by at most 2^-39 of it below.  The SwiGLU rows likewise, rounded from
// float32 to fp16's 11 bits, because the products take both operands in fp16: off by at most 2^-11 of a value (an eighth
// of the bf16 result's rounding), or 2^-39 of the largest of its share for values more than 2^28 below that.
// ------------------------------------------------------------------------------------------------
constexpr int kWarps = 16;                   // that multiply
constexpr int kSumWarps = 4;                 // that add the warps' partial sums up and finish the rows
constexpr int kMainThreads = 32 * kWarps;
constexpr int kThreads = kMainThreads + 32 * kSumWarps;
constexpr int kBufs = kSumWarps;             // items whose partial sums may be waiting, one per summing warp
constexpr int kSlotBytes = 2560;             // per warp: two pieces of two 16-byte codes and 8 scale bytes a lane
constexpr int kCols = 2;                     // tokens of an entry at most
constexpr int kMaxEntries = 256;             // (expert, token group) pairs: at most one per route
constexpr int kMaxRoutes = 256;
constexpr int kLogitExperts = 2;             // experts a CTA scores at a time, by kLogitShares warps each
constexpr int kLogitShares = kThreads / 32 / kLogitExperts;
constexpr uint64_t kBarrierLimitNs = 2000000000ull;

struct FewShared {
  uint4 zero;
  uint16_t ent_expert[kMaxEntries];
  int16_t ent_route[kMaxEntries][kCols];     // column -> route, or -1
  float ent_w[kMaxEntries][kCols];           // column -> weight
  uint32_t route_expert[kMaxRoutes];
  float route_w[kMaxRoutes];
  uint8_t route_token[kMaxRoutes];
  uint32_t used[kFewMaxRows];                // slots of a token that own a result row
  uint32_t act_amax[kWarps][kCols];          // by warp along K and column
  uint32_t x_amax[kFewMaxRows];
  float x_inv[kFewMaxRows];                  // undoes the power of two of a row
  float logit_part[kLogitExperts][kLogitShares][kFewMaxRows];
  uint64_t full[kBufs], empty[kBufs];
  int warp_count[kThreads / 32];
  int entries, distinct, bad;
  int short_row;                             // a row has fewer finite scores than slots
  uint32_t abort;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory"); }

// Eight E2M1 codes -> four fp16 pairs, in order.
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&d)[4]) {
  asm("{\n\t.reg .b8 x0, x1, x2, x3;\n\t"
      "mov.b32 {x0, x1, x2, x3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, x0;\n\tcvt.rn.f16x2.e2m1x2 %1, x1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, x2;\n\tcvt.rn.f16x2.e2m1x2 %3, x3;\n\t}"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(w));
}
// Four E4M3 bytes -> float32.
__device__ __forceinline__ void e4m3x4_to_f32(uint32_t four, float (&f)[4]) {
  uint32_t lo, hi;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(four));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same from zero.
__device__ __forceinline__ void mma16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// All CTAs of the grid (co-resident: cooperative launch).  The arrivals of one barrier add up to 2^31: every CTA
// adds one, the first what is missing.  So the top bit flips when the last has come, and nothing has to be
// reset.  Thread 0 knows the bit from before its first arrival (it cannot flip without it), so an arrival needs no
// answer.  Arriving and waiting are apart, so that work may lie between them; false when the wait ran out.
// CTAs that gave up arrive no more, so the count is then short and a later call could pass a barrier early.  They
// leave that in the word behind the count (kCntFewExpired), and every call that finds it set does nothing until the
// layer's check has reported it and cleared both.
__device__ __forceinline__ uint32_t grid_bit(const uint32_t* count, uint32_t& expired) {
  uint32_t now;
  asm volatile("ld.relaxed.gpu.global.v2.u32 {%0, %1}, [%2];" : "=r"(now), "=r"(expired) : "l"(count) : "memory");
  return now & 0x80000000u;
}
__device__ __forceinline__ void grid_arrive(uint32_t* count) {
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t add = blockIdx.x == 0 ? 0x80000000u - (gridDim.x - 1) : 1u;
    asm volatile("red.release.gpu.global.add.u32 [%0], %1;" ::"l"(count), "r"(add) : "memory");
  }
}
__device__ bool grid_wait(uint32_t* count, uint32_t& bit, volatile uint32_t* abort) {
  if (threadIdx.x == 0) {
    uint64_t t0 = 0;
    for (uint32_t spin = 1;; ++spin) {
      uint32_t now;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(count) : "memory");
      if ((bit ^ now) >> 31) break;
      if ((spin & 255u) == 0u) {
        const uint64_t t = tc::global_timer_ns();
        if (t0 == 0) t0 = t;
        else if (t - t0 > kBarrierLimitNs) { *abort = 1u; break; }
      }
    }
  }
  bit ^= 0x80000000u;
  __syncthreads();
  return *abort == 0u;
}
__device__ __forceinline__ bool grid_barrier(uint32_t* count, uint32_t& bit, volatile uint32_t* abort) {
  grid_arrive(count);
  return grid_wait(count, bit, abort);
}

// A CTA's share of one of the two weight passes.  How an item of rows is shared by the warps (FewPass: kw along K,
// rw along the rows) follows from the shape alone, so that a row's sums do not depend on its batch.
struct Share { int begin, end, entry, first; };        // items, and the first one's entry and place in it
__device__ __forceinline__ Share share_of(const FewArgs& a, const FewPass& p, int entries) {
  const uint32_t items = static_cast<uint32_t>(entries) * p.per_entry;
  // items * i / grid without a division: a.grid_step is 2^32 / grid, rounded up, so the last share is cut at `items`
  auto border = [&](uint32_t i) {
    return min(items, static_cast<uint32_t>((static_cast<uint64_t>(items) * min(static_cast<uint64_t>(i) * a.grid_step, uint64_t{1} << 32)) >> 32));
  };
  Share s;
  s.begin = static_cast<int>(border(blockIdx.x));
  s.end = static_cast<int>(border(blockIdx.x + 1));
  s.entry = static_cast<int>(__umulhi(static_cast<uint32_t>(s.begin), p.per_entry_inv));    // begin / per_entry (few_pass)
  s.first = s.begin - s.entry * p.per_entry;
  return s;
}
// First row of a row unit: rows R .. R+7 and R+32 .. R+39 of a 128-row scale tile, whose scales lie
// next to each other in pairs (sf_tile_offset).  Units 2v and 2v+1 are 8 rows apart.
__device__ __forceinline__ int unit_row(int u) { return (u >> 3) * 128 + ((u >> 2) & 1) * 64 + (u & 3) * 8; }

// The warp's stream of slots: its K units of each item in turn, through both passes.  Everything but the two lane
// offsets is the same for the whole warp.
struct Stream {
  const uint8_t *codes, *sf;          // of the next slot
  const uint8_t *codes0, *sf0;        // of the pass, at this warp's first unit
  size_t second, sf_second;           // from a slot's first piece to its second
  uint32_t lane_codes, lane_low, lane_sf;      // this lane's place in a piece: rows g and g + 32, scales
  int row_bytes, rows, units, kw, kwi, rw, rwi, per_entry, shift;
  int k, u, j, left;                  // K unit, item within its entry, entry, items left (0: nothing more)
  uint32_t ring, head, ring_end;      // shared addresses, this lane's 16 bytes included

  __device__ __forceinline__ void begin_pass(const FewArgs& a, const FewShared& sh, const FewPass& p, const Share& s, bool gate_up,
                                             int warp, int lane) {
    const int g = lane >> 2, t = lane & 3;
    units = p.units; kw = p.kw; rw = kWarps / p.kw; per_entry = p.per_entry;
    kwi = warp & (kw - 1); rwi = warp >> p.log_kw;
    shift = gate_up ? 0 : 1;
    row_bytes = (gate_up ? a.hidden : a.inter) / 2;
    rows = gate_up ? a.inter : a.hidden;
    second = gate_up ? static_cast<size_t>(a.up_codes - a.gate_codes) : static_cast<size_t>(8) * row_bytes;
    sf_second = gate_up ? static_cast<size_t>(a.up_sf - a.gate_sf) : 128;
    lane_codes = static_cast<uint32_t>(g) * row_bytes + t * 16;
    lane_low = lane_codes + 32u * row_bytes;
    lane_sf = (t & 1) * 512 + g * 16;          // the four blocks this lane scales (multiply_slot)
    codes0 = (gate_up ? a.gate_codes : a.down_codes) + kwi * 64;
    sf0 = (gate_up ? a.gate_sf : a.down_sf) + kwi * 1024;
    left = kwi < units ? s.end - s.begin : 0;
    j = s.entry;
    u = s.first;
    if (left > 0) open(sh);
  }
  __device__ __forceinline__ void open(const FewShared& sh) {
    const int unit = (u * rw + rwi) << shift;
    const uint32_t expert = __shfl_sync(0xffffffffu, static_cast<uint32_t>(sh.ent_expert[j]), 0);
    const uint32_t row = expert * static_cast<uint32_t>(rows) + unit_row(unit);     // < 2^32: experts * rows
    codes = codes0 + static_cast<size_t>(row) * row_bytes;
    sf = sf0 + static_cast<size_t>(row >> 7) * (row_bytes >> 5) * 512 + (unit & 3) * 128 + ((unit >> 2) & 1) * 8;
    k = kwi;
  }
  __device__ __forceinline__ void issue(const FewShared& sh, int lane) {
    if (left > 0) {
      cp_async16(head, codes + lane_codes);
      cp_async16(head + 512, codes + lane_low);
      cp_async16(head + 1024, codes + second + lane_codes);
      cp_async16(head + 1536, codes + second + lane_low);
      cp_async8(head + 2048 - lane * 8, sf + lane_sf);
      cp_async8(head + 2304 - lane * 8, sf + sf_second + lane_sf);
      k += kw;
      codes += kw * 64;
      sf += kw * 1024;
      if (k >= units && --left > 0) {
        if (++u == per_entry) { u = 0; ++j; }
        open(sh);
      }
    }
    head += kSlotBytes;
    if (head == ring_end) head = ring;
    cp_async_commit();        // one group per call, also when nothing is left: the count of pending groups stays exact
  }
};

__device__ __forceinline__ void lds128(uint32_t (&v)[4], uint32_t at) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
}
// acc[m] += piece m's rows (g, g + 32) times the unit's columns, as far as this lane holds them: of token t / 2 (lane
// t of the row's four), blocks 4 (t & 1) .. + 3.  `slot`: shared address of the slot, this lane's 16 bytes included;
// `scales`: of the scale words of those blocks of rows g and g + 32, piece 0 (piece 1: 256 further).  The four sums (two
// pieces, two blocks a lane) are chains of products side by side.
__device__ __forceinline__ void multiply_slot(float (&acc)[2][2], uint32_t slot, uint32_t scales, const uint32_t (&b)[16]) {
  uint32_t w[4][4];           // piece 0 rows g, g + 32; piece 1 the same
#pragma unroll
  for (int i = 0; i < 4; ++i) lds128(w[i], slot + i * 512);
  uint32_t s[2][2];
#pragma unroll
  for (int m = 0; m < 2; ++m)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(s[m][0]), "=r"(s[m][1]) : "r"(scales + m * 256) : "memory");
  float c[2][2][4];           // [piece][first or second block of each lane]
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int i = 2 * half; i < 2 * half + 2; ++i) {
        uint32_t d0[4], d1[4];
        e2m1x8_to_f16(w[2 * m][i], d0);
        e2m1x8_to_f16(w[2 * m + 1][i], d1);
        if (i == 2 * half) mma16816_first(c[m][half], d0[0], d1[0], d0[1], d1[1], b[4 * i], b[4 * i + 1]);
        else mma16816(c[m][half], d0[0], d1[0], d0[1], d1[1], b[4 * i], b[4 * i + 1]);
        mma16816(c[m][half], d0[2], d1[2], d0[3], d1[3], b[4 * i + 2], b[4 * i + 3]);
      }
    }
  // columns 2t and 2t + 1 are lanes t' = 2 (t & 1) and the next: their first blocks are the word's bytes 0 and 2
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float f[4];
      e4m3x4_to_f32(s[m][r], f);
      acc[m][r] = fmaf(c[m][0][2 * r], f[0], acc[m][r]);
      acc[m][r] = fmaf(c[m][1][2 * r], f[1], acc[m][r]);
      acc[m][r] = fmaf(c[m][0][2 * r + 1], f[2], acc[m][r]);
      acc[m][r] = fmaf(c[m][1][2 * r + 1], f[3], acc[m][r]);
    }
}

// Power of two that brings a largest magnitude with these bits into [2^14, 2^15), and its inverse.
// Zero, infinite and NaN maxima: 1.  Far below 2^-112 the largest factor, 2^126, is kept.
__device__ __forceinline__ float f16_factor(uint32_t amax, float* inverse) {
  if (amax == 0u || amax >= 0x7f800000u) {
    *inverse = 1.0f;
    return 1.0f;
  }
  const int e = max(static_cast<int>(amax >> 23), 1) - 127;
  const int k = min(14 - e, 126);
  *inverse = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
  return __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
}

// Barrier of the multiplying warps alone.
__device__ __forceinline__ void main_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kMainThreads) : "memory"); }

// Columns of `cols` tokens, as fp16 in the order the lanes read them: [unit][quarter i][column][t] pieces of
// 16 B, piece (i, t) of a unit = its columns 32t + 8i .. + 7.
// The hidden rows' power of two is the row's (x_amax).
__device__ void load_hidden_columns(const FewArgs& a, const FewShared& sh, uint8_t* dst, int entry, int cols, bool identity) {
  const int k = a.hidden, per_col = k / 8;
  main_sync();                           // the previous columns have been read
  for (int c = 0; c < cols; ++c) {
    int tok = c;
    if (!identity) {
      const int route = sh.ent_route[entry][c];
      if (route < 0) continue;           // nobody reads the column's results
      tok = sh.route_token[route];
    }
    float inv;
    const float f = f16_factor(sh.x_amax[tok], &inv);
    for (int o = threadIdx.x; o < per_col; o += kMainThreads) {       // 8-value pieces of the row
      const int unit = o >> 4, t = (o >> 2) & 3, q = o & 3;
      const uint4 x = *reinterpret_cast<const uint4*>(a.hidden_rows + static_cast<size_t>(tok) * k + o * 8);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      uint32_t h[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const __half2 p = __floats2half2_rn(__uint_as_float(w[n] << 16) * f, __uint_as_float(w[n] & 0xffff0000u) * f);
        h[n] = *reinterpret_cast<const uint32_t*>(&p);
      }
      *reinterpret_cast<uint4*>(dst + ((unit * 4 + q) * cols * 4 + c * 4 + t) * static_cast<size_t>(16)) = make_uint4(h[0], h[1], h[2], h[3]);
    }
  }
  main_sync();
}
// The SwiGLU rows' is that of the units one warp adds up (units kw apart): they alone share an accumulator.
__device__ void load_act_columns(const FewArgs& a, FewShared& sh, uint8_t* dst, int entry, int cols, int kw) {
  const int k = a.inter, per_col = k / 8;
  main_sync();
  for (int i = threadIdx.x; i < kWarps * kCols; i += kMainThreads) sh.act_amax[i / kCols][i % kCols] = 0u;
  main_sync();
  auto read = [&](int route, int o, float (&v)[8]) {
    const float4* src = reinterpret_cast<const float4*>(a.act + static_cast<size_t>(route) * k + o * 8);
    const float4 x = __ldcg(src), y = __ldcg(src + 1);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
  };
  const int pieces = cols * per_col;
  const bool keep = pieces <= kMainThreads;      // a piece a thread: read once
  float v[8];
  for (int i = threadIdx.x; i < pieces; i += kMainThreads) {        // a unit is 16 neighbouring lanes (k % 256 == 0)
    const int c = i / per_col, o = i - c * per_col, route = sh.ent_route[entry][c];
    uint32_t m = 0u;
    if (route >= 0) {
      read(route, o, v);
#pragma unroll
      for (int n = 0; n < 8; ++n) m = max(m, __float_as_uint(v[n]) & 0x7fffffffu);
    }
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, s));
    if ((threadIdx.x & 15) == 0) atomicMax(&sh.act_amax[(o >> 4) & (kw - 1)][c], m);
  }
  main_sync();
  for (int i = threadIdx.x; i < pieces; i += kMainThreads) {
    const int c = i / per_col, o = i - c * per_col, route = sh.ent_route[entry][c];
    if (route < 0) continue;
    const int unit = o >> 4, t = (o >> 2) & 3, q = o & 3;
    float inv;
    if (!keep) read(route, o, v);
    const float f = f16_factor(sh.act_amax[unit & (kw - 1)][c], &inv);
    uint32_t h[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const __half2 p = __floats2half2_rn(v[2 * n] * f, v[2 * n + 1] * f);
      h[n] = *reinterpret_cast<const uint32_t*>(&p);
    }
    *reinterpret_cast<uint4*>(dst + ((unit * 4 + q) * cols * 4 + c * 4 + t) * static_cast<size_t>(16)) = make_uint4(h[0], h[1], h[2], h[3]);
  }
  main_sync();
}

// Lane (g, t) holds the values of lane t in product column g = 4 token + t': they are the token's where t' = t, else
// zero (read from FewShared::zero, with a step of nothing).
__device__ __forceinline__ void load_b(uint32_t (&b)[16], uint32_t lane_columns, int unit, uint32_t lane_step) {
  const uint32_t at = lane_columns + unit * 4 * lane_step;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t q[4];
    lds128(q, at + i * lane_step);
    b[4 * i] = q[0]; b[4 * i + 1] = q[1]; b[4 * i + 2] = q[2]; b[4 * i + 3] = q[3];
  }
}

// Partial sums of an item: [warp][piece m][row][column], times what undoes the power of two of the column.  Two lanes
// share a token.
__device__ __forceinline__ void store_partial(float* red, const float (&acc)[2][2], float factor, int lane, int cols) {
  const int g = lane >> 2, c = (lane & 3) >> 1;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float v = (acc[m][r] + __shfl_xor_sync(0xffffffffu, acc[m][r], 1)) * factor;
      if ((lane & 1) == 0 && c < cols) red[(m * 16 + r * 8 + g) * cols + c] = v;
    }
}

// Top-k of one row by one warp: the largest keys, the lower id first among equal ones.  Slots that no key is left
// for name expert 0 with weight 0, as in the router (router.cu); such a row may name it more than once.
template <int kKeys>
__device__ __forceinline__ void select_row(const FewArgs& a, FewShared& sh, int row, int lane) {
  uint2 v[kKeys];            // key, score
#pragma unroll
  for (int i = 0; i < kKeys; ++i)
    v[i] = lane + 32 * i < a.experts ? __ldcg(a.scores + row * a.experts + lane + 32 * i) : make_uint2(0u, 0u);
  float sum = 0.0f, my_score = 0.0f;
  uint32_t mine = 0;
#pragma unroll 1
  for (int s = 0; s < a.top_k; ++s) {
    uint32_t best[kKeys];
#pragma unroll
    for (int i = 0; i < kKeys; ++i) best[i] = v[i].x;
#pragma unroll
    for (int h = kKeys / 2; h > 0; h /= 2)
#pragma unroll
      for (int i = 0; i < h; ++i) best[i] = max(best[i], best[i + h]);
    const uint32_t top = __reduce_max_sync(0xffffffffu, best[0]);
    uint32_t id = 0xffffffffu, score = 0u;
#pragma unroll
    for (int i = kKeys - 1; i >= 0; --i)
      if (v[i].x == top) { id = lane + 32 * i; score = v[i].y; }
    const uint32_t first = top != 0u ? __reduce_min_sync(0xffffffffu, id) : kNoRoute;
    const float chosen = top != 0u ? __uint_as_float(__shfl_sync(0xffffffffu, score, first & 31)) : 0.0f;
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
      if (lane + 32 * i == static_cast<int>(first)) v[i].x = 0u;
    sum += chosen;
    if (lane == s) { mine = first; my_score = chosen; }
  }
  if (lane < a.top_k) {
    const int r = row * a.top_k + lane;
    const bool none = mine == kNoRoute;
    if (none) sh.short_row = 1;
    sh.route_expert[r] = none ? 0u : mine;
    sh.route_w[r] = my_score * (a.scaling / fmaxf(sum, 1e-12f));
  }
}

// Routes of all rows, then the list of entries (sh.ent_*).  `scratch`: for every expert a word and a half-word.
__device__ void route_and_select(const FewArgs& a, FewShared& sh, uint8_t* scratch, bool identity) {
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int routes = a.rows * a.top_k;
  uint32_t* mask = reinterpret_cast<uint32_t*>(scratch);                            // rows that name an expert
  uint16_t* first_entry = reinterpret_cast<uint16_t*>(mask + a.experts);            // [expert]
  for (int i = tid; i < a.experts; i += kThreads) mask[i] = 0u;
  for (int i = tid; i < routes * kCols; i += kThreads) {    // at most one entry per route
    sh.ent_route[i / kCols][i % kCols] = -1;
    sh.ent_w[i / kCols][i % kCols] = 0.0f;
  }
  if (tid < kFewMaxRows) sh.used[tid] = 0u;
  if (tid == 0) { sh.bad = 0; sh.distinct = 0; }
  if (a.scores != nullptr) {
    if (warp < a.rows) {
      if (a.experts <= 256) select_row<8>(a, sh, warp, lane);
      else select_row<32>(a, sh, warp, lane);
    }
  } else if (tid < routes) {
    sh.route_expert[tid] = a.topk_idx[tid];
    sh.route_w[tid] = a.topk_w[tid];
  }
  __syncthreads();
  // Entries, in the order of the first route that names each: an expert's rows in groups of kCols
  // (identity: all rows are one group and a row's column is its number).
  const bool search = a.scores == nullptr || sh.short_row != 0;      // else the selection names nobody twice
  uint32_t e = kNoRoute;
  int slot = 0, token = 0;
  bool live = false;
  float w = 0.0f;
  if (tid < routes) {
    e = sh.route_expert[tid];
    w = sh.route_w[tid];
    token = tid / a.top_k; slot = tid - token * a.top_k;
    sh.route_token[tid] = static_cast<uint8_t>(token);
    live = e < static_cast<uint32_t>(a.experts);
    if (!live && e != kNoRoute) sh.bad = 1;
    const uint32_t* row = sh.route_expert + token * a.top_k;
    for (int s = 0; s < a.top_k && search; ++s) {
      if (s == slot || row[s] != e) continue;
      if (s < slot) live = false;                 // the row has named this expert before: its weight went there
      else w += sh.route_w[token * a.top_k + s];
    }
    if (blockIdx.x == 0) {                        // either may be wanted alone
      if (a.out_idx != nullptr) a.out_idx[tid] = e;
      if (a.out_w != nullptr) a.out_w[tid] = sh.route_w[tid];
    }
    if (live) {
      atomicOr(&mask[e], 1u << token);
      atomicOr(&sh.used[token], 1u << slot);
    }
  }
  __syncthreads();
  // An expert's entries follow each other, so that their passes over its weights run side by side and meet in the L2.
  const uint32_t rows_of = live ? mask[e] : 0u;
  const int rank = __popc(rows_of & ((1u << token) - 1u));
  const int opens = !live || rank != 0 ? 0 : identity ? 1 : (__popc(rows_of) + kCols - 1) / kCols;      // entries from here
  int upto = opens;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sh.warp_count[warp] = upto;
  __syncthreads();
  int before = upto - opens, total = 0;
#pragma unroll
  for (int i = 0; i < kMaxRoutes / 32; ++i) {
    if (i < warp) before += sh.warp_count[i];
    total += sh.warp_count[i];
  }
  if (opens > 0) {
    first_entry[e] = static_cast<uint16_t>(before);
    atomicAdd(&sh.distinct, 1);
  }
  if (tid == 0) sh.entries = total;
  __syncthreads();
  if (live) {
    const int entry = first_entry[e] + (identity ? 0 : rank / kCols), col = identity ? token : rank % kCols;
    sh.ent_expert[entry] = static_cast<uint16_t>(e);
    sh.ent_route[entry][col] = static_cast<int16_t>(tid);
    sh.ent_w[entry][col] = w;
  }
  __syncthreads();
}

// Logits of all rows, kLogitExperts experts of this CTA at a time: every warp one expert and one share of the
// columns, the shares added in order.  (Complete logits in one place: adding partial ones from every CTA would cost
// the selection an access to the L2 each.)
__device__ void score_experts(const FewArgs& a, FewShared& sh, int warp, int lane) {
  const int half = warp / kLogitShares, share = warp - half * kLogitShares, units = a.hidden / 128;
  const int u0 = units * share / kLogitShares, u1 = units * (share + 1) / kLogitShares;
#pragma unroll 1
  for (int e0 = blockIdx.x; e0 < a.experts; e0 += kLogitExperts * gridDim.x) {
    const int e_mine = e0 + half * gridDim.x;
    const float* wrow = a.router_w + static_cast<size_t>(e_mine) * a.hidden + lane * 4;
#pragma unroll 1
    for (int t0 = 0; t0 < a.rows && e_mine < a.experts; t0 += 4) {
      const uint16_t* xrow = a.hidden_rows + static_cast<size_t>(t0) * a.hidden + lane * 4;
      float acc[4] = {};
#pragma unroll 1
      for (int ub = u0; ub < u1; ub += 5) {            // five units of four rows in flight
        float4 w[5];
        uint2 x[4][5];
#pragma unroll
        for (int i = 0; i < 5; ++i) {
          const bool in = ub + i < u1;
          w[i] = in ? __ldg(reinterpret_cast<const float4*>(wrow + (ub + i) * 128)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int t = 0; t < 4; ++t)
            x[t][i] = in && t0 + t < a.rows ? __ldg(reinterpret_cast<const uint2*>(xrow + static_cast<size_t>(t) * a.hidden + (ub + i) * 128))
                                            : make_uint2(0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < 5; ++i)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            if (ub + i >= u1) continue;                // (zero times a weight that is not finite)
            acc[t] = fmaf(__uint_as_float(x[t][i].x << 16), w[i].x, acc[t]);
            acc[t] = fmaf(__uint_as_float(x[t][i].x & 0xffff0000u), w[i].y, acc[t]);
            acc[t] = fmaf(__uint_as_float(x[t][i].y << 16), w[i].z, acc[t]);
            acc[t] = fmaf(__uint_as_float(x[t][i].y & 0xffff0000u), w[i].w, acc[t]);
          }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float s = warp_sum(acc[t]);
        if (lane == 0) sh.logit_part[half][share][t0 + t] = s;
      }
    }
    __syncthreads();
    const int h = threadIdx.x / kFewMaxRows, t = threadIdx.x % kFewMaxRows;
    const int e = e0 + h * static_cast<int>(gridDim.x);
    if (h < kLogitExperts && t < a.rows && e < a.experts) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < kLogitShares; ++i) s += sh.logit_part[h][i][t];
      // a key that orders like score + bias and the score; zero, as for no expert, where they are not finite: the
      // router picks none of those (a finite value's key is at least 2^23)
      const float score = sigmoid_f32(s), rank = score + __ldg(a.router_b + e);
      const uint32_t u = __float_as_uint(rank == 0.0f ? 0.0f : rank);
      a.scores[t * a.experts + e] = make_uint2(!isfinite(rank) ? 0u : ((u >> 31) ? ~u : u | 0x80000000u), __float_as_uint(score));
    }
    __syncthreads();
  }
}

template <int kRing>
__global__ void __launch_bounds__(kThreads, 1) few_layer_kernel(FewArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  FewShared& sh = *reinterpret_cast<FewShared*>(smem);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid / 32, 0), lane = tid % 32;
  const int cols = min(a.rows, kCols);
  const bool identity = a.rows <= kCols;
  uint8_t* ring = smem + ((sizeof(FewShared) + 127) & ~static_cast<size_t>(127));
  float* red = reinterpret_cast<float*>(ring + kRing * kWarps * kSlotBytes);
  const int red_floats = kWarps * 32 * cols;
  uint8_t* columns = reinterpret_cast<uint8_t*>(red + kBufs * red_floats);
  if (tid == 0) {
    sh.abort = 0u;
    sh.short_row = 0;
    sh.zero = make_uint4(0u, 0u, 0u, 0u);
    for (int i = 0; i < kBufs; ++i) {
      tc::mbar_init(&sh.full[i], kWarps);
      tc::mbar_init(&sh.empty[i], 1);
    }
  }
  if (tid < kFewMaxRows) sh.x_amax[tid] = 0u;
  __syncthreads();

  uint32_t expired = 0u, bit = tid == 0 ? grid_bit(a.sync, expired) : 0u;
  if (a.scores != nullptr) {
    score_experts(a, sh, warp, lane);
    grid_arrive(a.sync);
  }
  if (expired != 0u) sh.abort = 1u;
  // the rows' largest magnitudes, 256 values a warp
  const int row_pieces = a.hidden / 256;
#pragma unroll 1
  for (int i = warp; i < a.rows * row_pieces; i += kThreads / 32) {
    const uint4 q = *reinterpret_cast<const uint4*>(a.hidden_rows + static_cast<size_t>(i) * 256 + lane * 8);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    uint32_t m = 0;
#pragma unroll
    for (int v = 0; v < 4; ++v) m = max(m, max((w[v] << 16) & 0x7fffffffu, w[v] & 0x7fff0000u));
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) atomicMax(&sh.x_amax[i / row_pieces], m);
  }
  __syncthreads();
  if (sh.abort != 0u) return;            // an earlier call's: nothing is written
  if (tid < a.rows) f16_factor(sh.x_amax[tid], &sh.x_inv[tid]);
  if (identity && warp < kWarps) load_hidden_columns(a, sh, columns, 0, cols, true);    // needs no routes
  if (a.scores != nullptr) {
    if (!grid_wait(a.sync, bit, &sh.abort)) {
      if (tid == 0) atomicOr(a.sync + 1, static_cast<uint32_t>(kErrWaitTimeout));
      return;
    }
  }
  route_and_select(a, sh, ring, identity);
  const int entries = __shfl_sync(0xffffffffu, sh.entries, 0);
  if (blockIdx.x == 0 && tid == 0) {
    a.error_word[0] = sh.bad ? static_cast<uint32_t>(kErrBadExpert) : 0u;
    a.counters[kCntChunks] = static_cast<uint32_t>(entries);
    a.counters[kCntDistinct] = static_cast<uint32_t>(sh.distinct);
  }

  const Share s1 = share_of(a, a.pass[0], entries), s2 = share_of(a, a.pass[1], entries);
  if (warp < kWarps) {
    // ---- the multiplying warps: the weight stream, then gate and up (pass 0) and down (pass 1) ----
    Stream st;
    st.ring = smem_addr(ring) + warp * kRing * kSlotBytes + lane * 16;
    st.ring_end = st.ring + kRing * kSlotBytes;
    st.head = st.ring;
    st.begin_pass(a, sh, a.pass[0], s1, true, warp, lane);
    bool first_pass = true;
    auto issue = [&] {
      if (st.left == 0 && first_pass) {
        st.begin_pass(a, sh, a.pass[1], s2, false, warp, lane);
        first_pass = false;
      }
      st.issue(sh, lane);
    };
#pragma unroll 1
    for (int i = 0; i < kRing - 1; ++i) issue();
    uint32_t tail = st.ring;
    const int lane_token = lane >> 4;                  // of the product column this lane brings, and whether it has values
    const bool mine = ((lane >> 2) & 3) == (lane & 3) && lane_token < cols;
    const uint32_t lane_columns = mine ? smem_addr(columns) + (lane_token * 4 + (lane & 3)) * 16 : smem_addr(&sh.zero);
    const uint32_t lane_step = mine ? cols * 64 : 0;
    const int scale_at = 2048 - lane * 8;
    uint32_t b[16];
    int n = 0;                     // items so far: buffer n % kBufs, its round n / kBufs
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
      if (pass == 1) grid_barrier(a.sync, bit, &sh.abort);
      const Share s = pass == 0 ? s1 : s2;
      const FewPass p = a.pass[pass];
      const int kwi = warp & (p.kw - 1);
      int entry = -1, j = s.entry, u = s.first;
      float factor = 1.0f;
#pragma unroll 1
      for (int it = s.begin; it < s.end; ++it) {
        if (j != entry) {
          if (pass == 0) {
            if (!identity) load_hidden_columns(a, sh, columns, j, cols, false);
          } else {
            load_act_columns(a, sh, columns, j, cols, p.kw);
            f16_factor(sh.act_amax[kwi][(lane & 3) >> 1], &factor);
          }
          entry = j;
        }
        float acc[2][2] = {};
#pragma unroll 1
        for (int k = kwi; k < p.units; k += p.kw) {
          load_b(b, lane_columns, k, lane_step);
          cp_async_wait<kRing - 2>();
          multiply_slot(acc, tail, tail + scale_at, b);
          tail += kSlotBytes;
          if (tail == st.ring_end) tail = st.ring;
          issue();
        }
        // The item's partial sums go to a summing warp.  A wait that ran out is seen by everybody at the grid's next
        // barrier; until then the warp keeps step with the others, which meet it at the barriers around their columns.
        const int buf = n % kBufs;
        const uint32_t empty_parity = ((n / kBufs) & 1) ^ 1u;
        if (__all_sync(0xffffffffu, tc::mbar_try_wait(&sh.empty[buf], empty_parity)) || tc::mbar_wait_warp(&sh.empty[buf], empty_parity, &sh.abort)) {
          store_partial(red + buf * red_floats + warp * 32 * cols, acc, factor, lane, cols);
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&sh.full[buf]);
        }
        ++n;
        if (++u == p.per_entry) { u = 0; ++j; }
      }
    }
    cp_async_wait<0>();
  } else {
    // ---- the summing warps: every kSumWarps-th item each, the warps' shares added in order ----
    const int mine = warp - kWarps;
    const float* part = red + mine * red_floats;
    bool alive = true;
    int base = 0;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
      const Share s = pass == 0 ? s1 : s2;
      const FewPass p = a.pass[pass];
      const int items = s.end - s.begin, rw = kWarps >> p.log_kw, warps_k = min(p.kw, p.units);
      // the CTA's item number base + i is this warp's when it is `mine` modulo kSumWarps
      int i = (mine - base % kSumWarps + kSumWarps) % kSumWarps;
      int u = s.first, j = s.entry, at = 0;          // entry and place of item `at`
#pragma unroll 1
      for (; i < items && alive; i += kSumWarps) {
        u += i - at;
        at = i;
        while (u >= p.per_entry) { u -= p.per_entry; ++j; }
        const float* s2p = a.scale2 + sh.ent_expert[j] * 3 + (pass == 0 ? lane >> 4 : 2);
        const float scale2 = __ldg(s2p);
        alive = tc::mbar_wait_warp(&sh.full[mine], ((base + i) / kBufs) & 1, &sh.abort);
        if (!alive) break;
#pragma unroll 1
        for (int q0 = 0; q0 < rw * kCols; q0 += 4) {   // four sums (row group, column) side by side
          float sum[4] = {};
          const float* src = part + ((q0 / kCols) * p.kw * 32 + lane) * cols;
#pragma unroll 2
          for (int w = 0; w < warps_k; ++w)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (q0 + x < rw * kCols && x % kCols < cols) sum[x] += src[((x / kCols) * p.kw + w) * 32 * cols + x % kCols];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int r = (q0 + x) / kCols, c = x % kCols;
            const int route = r < rw && c < cols ? sh.ent_route[j][c] : -1;
            if (route < 0) continue;
            if (pass == 0) {                           // lanes 0..15 gate, 16..31 up
              const float v = sum[x] * (scale2 * sh.x_inv[sh.route_token[route]]);
              const float up = __shfl_down_sync(0xffffffffu, v, 16);
              if (lane < 16)
                a.act[static_cast<size_t>(route) * a.inter + unit_row(u * rw + r) + (lane & 7) + (lane >> 3) * 32] =
                    sh.ent_w[j][c] * (__fdividef(v, 1.0f + __expf(-v)) * up);
            } else {
              a.route_out[static_cast<size_t>(route) * a.hidden + unit_row((u * rw + r) * 2 + (lane >> 4)) + (lane & 7) +
                          ((lane >> 3) & 1) * 32] = sum[x] * scale2;
            }
          }
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sh.empty[mine]);
      }
      base += items;
      if (pass == 0) grid_barrier(a.sync, bit, &sh.abort);
    }
  }
  if (!grid_barrier(a.sync, bit, &sh.abort)) {
    if (tid == 0) atomicOr(a.sync + 1, static_cast<uint32_t>(kErrWaitTimeout));
    return;
  }

  // ---- combine ----
  const int values = a.rows * a.hidden;
  for (int i = blockIdx.x * kThreads + tid; i < values; i += gridDim.x * kThreads) {
    const int t = i / a.hidden, h = i - t * a.hidden;
    float y = 0.0f;
    const uint32_t used = sh.used[t];
    const float* src = a.route_out + static_cast<size_t>(t) * a.top_k * a.hidden + h;
#pragma unroll 8
    for (int s = 0; s < a.top_k; ++s)
      if (used >> s & 1u) y += __ldcg(src + static_cast<size_t>(s) * a.hidden);
    if (a.shared != nullptr) y += bf16_bits_to_f32(a.shared[i]);
    if (a.residual != nullptr) y += bf16_bits_to_f32(a.residual[i]);
    a.out[i] = f32_to_bf16_rne(y);
  }
}

// Verification form: one warp per (route, intermediate row).
__global__ void few_fc1_simt_kernel(FewArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int route = blockIdx.y, token = route / a.top_k, lane = threadIdx.x % 32;
  const int m = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (m >= a.inter) return;
  const uint32_t e = a.topk_idx[route];
  float* dst = a.act + static_cast<size_t>(route) * a.inter + m;
  if (e >= static_cast<uint32_t>(a.experts)) {
    if (lane == 0) {
      *dst = 0.0f;
      if (e != kNoRoute) atomicOr(a.error_word, static_cast<uint32_t>(kErrBadExpert));
    }
    return;
  }
  const size_t row = static_cast<size_t>(e) * a.inter + m;
  const uint16_t* x = a.hidden_rows + static_cast<size_t>(token) * a.hidden;
  float g = 0.0f, u = 0.0f;
  for (int j = lane; j < a.hidden / 16; j += 32) {
    const uint8_t* cg = a.gate_codes + row * (a.hidden / 2) + j * 8;
    const uint8_t* cu = a.up_codes + row * (a.hidden / 2) + j * 8;
    float sg = 0.0f, su = 0.0f;
    for (int i = 0; i < 16; ++i) {
      const float xv = bf16_bits_to_f32(x[j * 16 + i]);
      sg = fmaf(xv, e2m1_to_f32((cg[i / 2] >> (4 * (i & 1))) & 15u), sg);
      su = fmaf(xv, e2m1_to_f32((cu[i / 2] >> (4 * (i & 1))) & 15u), su);
    }
    const size_t so = sf_tile_offset(row, j, a.hidden / 16);
    g = fmaf(sg, e4m3_to_f32(a.gate_sf[so]), g);
    u = fmaf(su, e4m3_to_f32(a.up_sf[so]), u);
  }
  g = warp_sum(g) * a.scale2[e * 3];
  u = warp_sum(u) * a.scale2[e * 3 + 1];
  if (lane == 0) *dst = a.topk_w[route] * (g / (1.0f + expf(-g)) * u);
}

// One warp per (token, hidden row).
__global__ void few_fc2_simt_kernel(FewArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int token = blockIdx.y, lane = threadIdx.x % 32;
  const int h = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (h >= a.hidden) return;
  float y = 0.0f;
  for (int s = 0; s < a.top_k; ++s) {
    const int route = token * a.top_k + s;
    const uint32_t e = a.topk_idx[route];
    if (e >= static_cast<uint32_t>(a.experts)) continue;
    const size_t row = static_cast<size_t>(e) * a.hidden + h;
    const float* act = a.act + static_cast<size_t>(route) * a.inter;
    float part = 0.0f;
    for (int j = lane; j < a.inter / 16; j += 32) {
      const uint8_t* c = a.down_codes + row * (a.inter / 2) + j * 8;
      float sum = 0.0f;
      for (int i = 0; i < 16; ++i) sum = fmaf(act[j * 16 + i], e2m1_to_f32((c[i / 2] >> (4 * (i & 1))) & 15u), sum);
      part = fmaf(sum, e4m3_to_f32(a.down_sf[sf_tile_offset(row, j, a.inter / 16)]), part);
    }
    y = fmaf(warp_sum(part), a.scale2[e * 3 + 2], y);
  }
  if (lane == 0) {
    const size_t at = static_cast<size_t>(token) * a.hidden + h;
    if (a.shared != nullptr) y += bf16_bits_to_f32(a.shared[at]);
    if (a.residual != nullptr) y += bf16_bits_to_f32(a.residual[at]);
    a.out[at] = f32_to_bf16_rne(y);
  }
}

}  // namespace

FewPass few_pass(int k, int groups) {
  FewPass p{};
  p.units = k / 128;
  p.kw = kWarps;
  p.log_kw = 4;
  while (p.kw > 2 && p.kw * 2 > p.units) {      // two units a warp or more, so that handing a sum over is rare
    p.kw /= 2;
    --p.log_kw;
  }
  p.per_entry = groups / (kWarps / p.kw);
  p.per_entry_inv = static_cast<uint32_t>(((uint64_t{1} << 32) + p.per_entry - 1) / p.per_entry);
  return p;
}

namespace {
size_t few_smem(int ring, int cols, int k) {
  const size_t fixed = (sizeof(FewShared) + 127) & ~static_cast<size_t>(127);
  return fixed + static_cast<size_t>(ring) * kWarps * kSlotBytes + static_cast<size_t>(kBufs) * kWarps * 32 * cols * 4 +
         static_cast<size_t>(cols) * k * 2;
}
constexpr size_t kSmemMost = 227 * 1024;

template <int kRing>
glmrt_status_t launch_ring(const FewArgs& a, size_t smem, int sm_count, cudaStream_t s) {
  static std::atomic<uint64_t> configured{0};
  GLMRT_RETURN_IF_ERROR(ensure_smem_limit(configured, few_layer_kernel<kRing>, kSmemMost, "cudaFuncSetAttribute(few_layer_kernel)"));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(sm_count));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  FewArgs args = a;
  args.grid_step = static_cast<uint32_t>(((uint64_t{1} << 32) + sm_count - 1) / sm_count);
  cudaError_t err = cudaLaunchKernelEx(&cfg, few_layer_kernel<kRing>, args);
  if (err != cudaSuccess) return fail_cuda(GLMRT_STATUS_COPY_FAILED, "few_layer_kernel", err);
  GLMRT_LAUNCH_CHECK("few_layer_kernel");
  return GLMRT_STATUS_OK;
}
}  // namespace

// What fits into shared memory decides the depth of the stream; the selection's scratch (6 bytes an expert) lies in
// its ring, and at least three slots are needed.  Whether it fits is asked for the widest entries, also where one row
// would do with less: a row's result must not depend on how many rows the call has.
bool few_fused_supported(const FewArgs& a) {
  static_assert(1024 * 6 <= 3 * kWarps * kSlotBytes, "selection scratch fits the ring");
  // (per_entry < 4096 makes the multiplication by its inverse exact: at most 256 entries)
  return few_smem(3, kCols, std::max(a.hidden, a.inter)) <= kSmemMost && a.experts <= 1024 && a.pass[0].per_entry > 1 &&
         a.pass[0].per_entry < 4096 && a.pass[1].per_entry > 1 && a.pass[1].per_entry < 4096;
}
glmrt_status_t launch_few_fused(const FewArgs& a, int sm_count, cudaStream_t s) {
  const size_t four = few_smem(4, std::min(a.rows, kCols), std::max(a.hidden, a.inter));
  if (four <= kSmemMost) return launch_ring<4>(a, four, sm_count, s);
  return launch_ring<3>(a, few_smem(3, std::min(a.rows, kCols), std::max(a.hidden, a.inter)), sm_count, s);
}

glmrt_status_t launch_few_simt(const FewArgs& a, cudaStream_t s) {
  launch_pdl(few_fc1_simt_kernel, dim3((a.inter + 7) / 8, a.rows * a.top_k), dim3(256), 0, s, a);
  GLMRT_LAUNCH_CHECK("few_fc1_simt_kernel");
  launch_pdl(few_fc2_simt_kernel, dim3((a.hidden + 7) / 8, a.rows), dim3(256), 0, s, a);
  GLMRT_LAUNCH_CHECK("few_fc2_simt_kernel");
  return GLMRT_STATUS_OK;
}

}  // namespace glmrt
