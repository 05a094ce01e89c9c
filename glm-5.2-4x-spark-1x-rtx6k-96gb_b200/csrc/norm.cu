// The boundary between two blocks of a layer in one pass over the rows:
//
//   d = delta                                       the finished block's output (optional)
//   d = d * rsqrt(mean(d^2) + eps) * post_weight    norm after the block (optional)
//   d = d * gate                                    per row, per channel or per value (optional)
//   r = residual + scale * d                        -> residual_out
//   y = r * rsqrt(mean(r^2) + eps) * norm_weight    -> normalized, the next block's input
//
// The sparse layer's own use is the plain form (no post norm, no gate, scale 1): attention's result
// joins the residual stream and the rows the router, the experts and the shared expert read come out
// normalised (python/reference/glmrt_reference/glm_moe_dsa_layer_ref.py:157-206).
//
// Arithmetic is float32 throughout; each output is rounded once (nearest even), and `y` is formed
// from the unrounded r, so it does not inherit the rounding of the stored residual.
//
// Bound by memory: each value is read once and written once and does about ten operations.  One row
// belongs to one group of threads that keeps all of it in registers (at most 32 values a thread)
// between the loads and the second statistic, so nothing is read twice.  Measured: 1 x 6144 bf16 2.3 to 2.8 us, 1021 x 4100
// float32 12.5 us = 5.4 TB/s, 8192 x 4096 float32 80 us = 6.7 TB/s, 8192 x 4100 bf16 56 us = 4.8 TB/s.
#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "tc_ptx.cuh"

namespace glmrt {
namespace {

constexpr int kMaxWidth = 32768;      // 1024 threads x 32 values

__device__ uint32_t g_norm_error;     // kErrWaitTimeout when a bounded wait ran out (glmrt_b200_operators_check)

struct NormArgs {
  const void *residual, *delta, *norm_w, *post_w, *gate;
  void *residual_out, *normalized;
  size_t residual_stride, delta_stride, gate_rs, gate_cs, residual_out_stride, normalized_stride;
  int rows, width;
  float scale, eps;
};

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<uint16_t>(uint16_t v) { return bf16_bits_to_f32(v); }
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ uint16_t from_f32<uint16_t>(float v) { return f32_to_bf16_rne(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }

// kVec consecutive values as they lie in memory: 16 or 8 aligned bytes, or one value.
template <typename T, int kVec>
struct alignas(kVec * sizeof(T)) Piece {
  T t[kVec];
  __device__ __forceinline__ static Piece load(const T* p) { return *reinterpret_cast<const Piece*>(p); }
  __device__ __forceinline__ void unpack(float (&v)[kVec]) const {
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = to_f32(t[i]);
  }
};
template <typename T, int kVec>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[kVec]) { Piece<T, kVec>::load(p).unpack(v); }
template <typename T, int kVec>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[kVec]) {
  Piece<T, kVec> q;
#pragma unroll
  for (int i = 0; i < kVec; ++i) q.t[i] = from_f32<T>(v[i]);
  *reinterpret_cast<Piece<T, kVec>*>(p) = q;
}
// Weights may be wider or narrower than the rows: kVec of them, at most 16 bytes a load.
template <typename W, int kVec>
__device__ __forceinline__ void load_weight(const W* p, float (&v)[kVec]) {
  constexpr int kPer = std::min<int>(16 / sizeof(W), kVec);
  if constexpr (kVec > 1) {
#pragma unroll
    for (int i = 0; i < kVec; i += kPer) {
      float t[kPer];
      load_vec<W, kPer>(p + i, t);
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[i + j] = t[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = to_f32(p[i]);
  }
}

// Sum over the threads of one row (blockDim.x of them); every thread gets it.
__device__ __forceinline__ float row_sum(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = blockDim.x / 32;
  if (warps == 1) return v;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  __syncthreads();                    // an earlier use of scratch has been read
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  v = lane < warps ? scratch[lane] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// T rows' type, W weights' type, kVec values per access, kNv accesses per thread.
template <typename T, typename W, int kVec, int kNv>
__global__ void __launch_bounds__(1024) block_norm_kernel(NormArgs a) {
  __shared__ float scratch[32];
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t row_i = blockIdx.x * blockDim.y + threadIdx.y;
  if (row_i >= static_cast<uint32_t>(a.rows)) return;        // blockDim.y > 1 only with one warp per row: whole warps leave
  const size_t row = static_cast<size_t>(row_i);
  const T* res = static_cast<const T*>(a.residual) + row * a.residual_stride;
  const float inv_width = 1.0f / static_cast<float>(a.width);
  auto column = [&](int n) { return (n * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * kVec; };
  // The residual is asked for with the branch, before the branch's statistic, where a thread has the
  // registers to hold it as it lies (widest float32 rows: after the statistic).
  constexpr bool kEarly = sizeof(T) * kVec * kNv <= 64;
  Piece<T, kVec> early[kEarly ? kNv : 1];
  if constexpr (kEarly) {
#pragma unroll
    for (int n = 0; n < kNv; ++n)
      if (column(n) < a.width) early[n] = Piece<T, kVec>::load(res + column(n));
  }
  float v[kNv][kVec];                 // the branch, then the new residual; zero past the width
  if (a.delta != nullptr) {
    const T* del = static_cast<const T*>(a.delta) + row * a.delta_stride;
#pragma unroll
    for (int n = 0; n < kNv; ++n) {
      if (column(n) < a.width) load_vec<T, kVec>(del + column(n), v[n]);
      else
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[n][i] = 0.0f;
    }
    if (a.post_w != nullptr) {
      float ss = 0.0f;
#pragma unroll
      for (int n = 0; n < kNv; ++n)
#pragma unroll
        for (int i = 0; i < kVec; ++i) ss += v[n][i] * v[n][i];
      const float rs = rsqrtf(row_sum(ss, scratch) * inv_width + a.eps);
#pragma unroll
      for (int n = 0; n < kNv; ++n) {
        if (column(n) >= a.width) continue;
        float w[kVec];
        load_weight<W, kVec>(static_cast<const W*>(a.post_w) + column(n), w);
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[n][i] *= rs * w[i];
      }
    }
    if (a.gate != nullptr) {
      const T* g = static_cast<const T*>(a.gate) + row * a.gate_rs;
#pragma unroll
      for (int n = 0; n < kNv; ++n) {
        if (column(n) >= a.width) continue;
        float s[kVec];
        if (a.gate_cs == 0) {
#pragma unroll
          for (int i = 0; i < kVec; ++i) s[i] = to_f32(*g);
        } else {
          load_vec<T, kVec>(g + column(n), s);
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[n][i] *= s[i];
      }
    }
  }
#pragma unroll
  for (int n = 0; n < kNv; ++n) {
    float r[kVec];
    if (column(n) < a.width) {
      if constexpr (kEarly) early[n].unpack(r);
      else load_vec<T, kVec>(res + column(n), r);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) r[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[n][i] = a.delta != nullptr ? fmaf(a.scale, v[n][i], r[i]) : r[i];
    if (a.delta != nullptr && column(n) < a.width)
      store_vec<T, kVec>(static_cast<T*>(a.residual_out) + row * a.residual_out_stride + column(n), v[n]);
  }
  float ss = 0.0f;
#pragma unroll
  for (int n = 0; n < kNv; ++n)
#pragma unroll
    for (int i = 0; i < kVec; ++i) ss += v[n][i] * v[n][i];
  const float rs = rsqrtf(row_sum(ss, scratch) * inv_width + a.eps);
  T* out = static_cast<T*>(a.normalized) + row * a.normalized_stride;
#pragma unroll
  for (int n = 0; n < kNv; ++n) {
    if (column(n) >= a.width) continue;
    float w[kVec];
    load_weight<W, kVec>(static_cast<const W*>(a.norm_w) + column(n), w);
#pragma unroll
    for (int i = 0; i < kVec; ++i) w[i] *= v[n][i] * rs;
    store_vec<T, kVec>(out + column(n), w);
  }
}

// Many wide bf16 rows: a CTA takes every gridDim-th row; bulk copies bring the next rows into a ring in shared
// memory while one is worked on, and the weights stay in registers (8192 x 6144: 71 us; four streams of 100 MB at the
// copy rate are 61).  Rows whose pieces are 16 bytes, aligned; two pieces a thread; no norm of the branch (its sum
// would make the chain of a row longer, and only two rows are under way on an SM).
template <typename W>
__global__ void __launch_bounds__(512, 2) block_norm_stream_kernel(NormArgs a, int stages, uint32_t row_bytes) {
  using T = uint16_t;
  constexpr int kVec = 8, kNv = 2, kPer = 16 / static_cast<int>(sizeof(W));
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float scratch[32];
  __shared__ uint64_t full[8];
  __shared__ uint32_t abort_word;
  volatile uint32_t* abort_flag = &abort_word;
  const bool branch = a.delta != nullptr;
  const uint32_t stage_bytes = row_bytes * (branch ? 2 : 1);
  if (threadIdx.x == 0) {
    abort_word = 0u;
    for (int i = 0; i < stages; ++i) tc::mbar_init(&full[i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  const uint64_t policy = tc::policy_evict_first();
  auto fetch = [&](int row, int stage) {
    const uint32_t at = tc::smem_u32(ring) + stage * stage_bytes;
    tc::mbar_expect_tx(&full[stage], stage_bytes);
    tc::bulk_load(at, static_cast<const T*>(a.residual) + static_cast<size_t>(row) * a.residual_stride, row_bytes, &full[stage], policy);
    if (branch)
      tc::bulk_load(at + row_bytes, static_cast<const T*>(a.delta) + static_cast<size_t>(row) * a.delta_stride, row_bytes, &full[stage], policy);
  };
  if (threadIdx.x == 0)
    for (int i = 0; i < stages; ++i) {
      const long long row = blockIdx.x + static_cast<long long>(i) * gridDim.x;
      if (row < a.rows) fetch(static_cast<int>(row), i);
    }
  const float inv_width = 1.0f / static_cast<float>(a.width);
  auto column = [&](int n) { return (n * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * kVec; };
  uint4 norm_w[kNv][kVec / kPer];
  auto take = [&](const void* w, uint4 (&q)[kVec / kPer], int c) {
#pragma unroll
    for (int i = 0; i < kVec / kPer; ++i) q[i] = *reinterpret_cast<const uint4*>(static_cast<const W*>(w) + c + i * kPer);
  };
  auto weight_at = [&](const uint4 (&q)[kVec / kPer], int i) { return to_f32(reinterpret_cast<const W*>(&q[i / kPer])[i % kPer]); };
#pragma unroll
  for (int n = 0; n < kNv; ++n)
    if (column(n) < a.width) take(a.norm_w, norm_w[n], column(n));
  int stage = 0;
  uint32_t phase = 0;
  for (long long row_i = blockIdx.x; row_i < a.rows; row_i += gridDim.x) {
    const size_t row = static_cast<size_t>(row_i);
    const bool valid = tc::mbar_wait_hot(&full[stage], phase, abort_flag);
    const T* res = reinterpret_cast<const T*>(ring + stage * stage_bytes);
    float v[kNv][kVec], r[kNv][kVec];
#pragma unroll
    for (int n = 0; n < kNv; ++n)
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[n][i] = r[n][i] = 0.0f;
#pragma unroll
    for (int n = 0; n < kNv; ++n)
      if (column(n) < a.width) {
        load_vec<T, kVec>(res + column(n), r[n]);
        if (branch) load_vec<T, kVec>(res + row_bytes / sizeof(T) + column(n), v[n]);
      }
    __syncthreads();                                    // everybody has its values: the stage may be filled again
    if (threadIdx.x == 0) {
      const long long next = row_i + static_cast<long long>(stages) * gridDim.x;
      if (next < a.rows) fetch(static_cast<int>(next), stage);
    }
    if (branch && a.gate != nullptr) {
      const T* g = static_cast<const T*>(a.gate) + row * a.gate_rs;
#pragma unroll
      for (int n = 0; n < kNv; ++n) {
        if (column(n) >= a.width) continue;
        float s[kVec];
        if (a.gate_cs == 0) {
#pragma unroll
          for (int i = 0; i < kVec; ++i) s[i] = to_f32(*g);
        } else {
          load_vec<T, kVec>(g + column(n), s);
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[n][i] *= s[i];
      }
    }
    float ss = 0.0f;
#pragma unroll
    for (int n = 0; n < kNv; ++n) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        v[n][i] = branch ? fmaf(a.scale, v[n][i], r[n][i]) : r[n][i];
        ss += v[n][i] * v[n][i];
      }
      if (branch && valid && column(n) < a.width)
        store_vec<T, kVec>(static_cast<T*>(a.residual_out) + row * a.residual_out_stride + column(n), v[n]);
    }
    const float rs = rsqrtf(row_sum(ss, scratch) * inv_width + a.eps);
#pragma unroll
    for (int n = 0; n < kNv; ++n)
      if (valid && column(n) < a.width) {
        float y[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) y[i] = weight_at(norm_w[n], i) * (v[n][i] * rs);
        store_vec<T, kVec>(static_cast<T*>(a.normalized) + row * a.normalized_stride + column(n), y);
      }
    if (++stage == stages) { stage = 0; phase ^= 1u; }
  }
  if (threadIdx.x == 0 && abort_word != 0u) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);    // let copies in flight land
    atomicOr(&g_norm_error, static_cast<uint32_t>(kErrWaitTimeout));
  }
}

template <typename T, typename W, int kVec, int kNv>
void launch(const NormArgs& a, int threads, cudaStream_t s) {
  const unsigned ty = threads == 32 ? 8 : 1;
  launch_pdl(block_norm_kernel<T, W, kVec, kNv>, dim3((static_cast<unsigned>(a.rows) + ty - 1) / ty),     // rows < 2^31
             dim3(static_cast<unsigned>(threads), ty), 0, s, a);
}

constexpr int kStreamRing = 104 * 1024;       // a CTA's rows in shared memory, two CTAs on an SM

template <typename W>
glmrt_status_t launch_stream(const NormArgs& a, int stages, uint32_t row_bytes, int ctas, cudaStream_t s) {
  static std::atomic<uint64_t> configured{0};
  GLMRT_RETURN_IF_ERROR(ensure_smem_limit(configured, block_norm_stream_kernel<W>, kStreamRing, "cudaFuncSetAttribute(block_norm_stream_kernel)"));
  const int pieces = a.width / 8;
  launch_pdl(block_norm_stream_kernel<W>, dim3(static_cast<unsigned>(ctas)), dim3(static_cast<unsigned>(((pieces + 1) / 2 + 31) / 32 * 32)),
             static_cast<size_t>(stages) * row_bytes * (a.delta != nullptr ? 2 : 1), s, a, stages, row_bytes);
  return GLMRT_STATUS_OK;
}

// Rows of one residual stream are at least this many values (8 MB of bf16) before bf16 rows are taken in 8-byte pieces.
constexpr long long kManyValues = 1ll << 22;

template <typename T, typename W, int kVec>
glmrt_status_t dispatch(const NormArgs& a, cudaStream_t s) {
  const int pieces = (a.width + kVec - 1) / kVec;
  constexpr int kMost = 32 / kVec;            // accesses per thread at 32 values
  constexpr bool kBf16 = sizeof(T) == 2;
  const bool many = static_cast<long long>(a.rows) * a.width >= kManyValues;
  if constexpr (kVec == 8) {
    // bf16 rows of 10 to 16 KB without a norm of the branch, at least four for each of the 296 CTAs (rows x width,
    // against the form below: 8192 x 6144 71 / 74 us, 8192 x 8192 93 / 106, 1200 x 8192 16.8 / 19.3; 8192 x 4096 55 / 52,
    // and with a norm of the branch 8192 x 6144 108 / 91).
    const uint32_t row_bytes = static_cast<uint32_t>(a.width) * sizeof(T);
    const int ctas = 2 * 148, stages = std::min<int>(8, kStreamRing / (row_bytes * (a.delta != nullptr ? 2 : 1)));
    if (a.post_w == nullptr && a.rows >= 4 * ctas && pieces >= 640 && pieces <= 1024) return launch_stream<W>(a, stages, row_bytes, ctas, s);
    // Many bf16 values: four pieces of 8 bytes a thread do better than two of 16 (with a norm of the branch, two / four:
    // 8192 x 2048 35 / 31 us, 8192 x 4096 75 / 64, 8192 x 6144 107 / 91, 8192 x 8192 156 / 132; but 1200 x 1024 4.0 / 4.7).
    if (many) return dispatch<T, W, 4>(a, s);
  }
  // A few rows: as many threads per row as it has pieces, for the latency.  More rows than SMs: two pieces a thread,
  // so that several rows share an SM and their loads overlap each other's reductions (measured at 333 x 5120 bf16
  // with both norms and a gate: one piece 5.9 us, two 5.1, four 8.9).
  int nv = 1;
  if (kBf16 && kVec == 4 && many) nv = 4;
  while (nv < kMost && (pieces + nv - 1) / nv > 1024) nv *= 2;
  if (a.rows > 2 * 148 && nv == 1 && pieces >= 256) nv = 2;
  const int threads = ((pieces + nv - 1) / nv + 31) / 32 * 32;
  if (nv == 1) launch<T, W, kVec, 1>(a, threads, s);
  else if (nv == 2) launch<T, W, kVec, 2>(a, threads, s);
  else if (nv == 4) launch<T, W, kVec, 4>(a, threads, s);
  if constexpr (kMost >= 8)
    if (nv == 8) launch<T, W, kVec, 8>(a, threads, s);
  if constexpr (kMost >= 32) {
    if (nv == 16) launch<T, W, kVec, 16>(a, threads, s);
    if (nv == 32) launch<T, W, kVec, 32>(a, threads, s);
  }
  return GLMRT_STATUS_OK;
}

// align: bytes that every row and weight piece may be read at once
template <typename T, typename W>
glmrt_status_t dispatch_vec(const NormArgs& a, int align, cudaStream_t s) {
  if (align == 16) return dispatch<T, W, 16 / static_cast<int>(sizeof(T))>(a, s);
  if constexpr (sizeof(T) == 2)
    if (align == 8) return dispatch<T, W, 4>(a, s);
  return dispatch<T, W, 1>(a, s);
}

struct Span { uintptr_t lo, hi; size_t stride; };
bool overlap(const Span& x, const Span& y) { return x.lo < y.hi && y.lo < x.hi; }

}  // namespace
}  // namespace glmrt

namespace glmrt {
glmrt_status_t norm_take_error(uint32_t* out) { return take_error_word(g_norm_error, out); }
}  // namespace glmrt

using namespace glmrt;

extern "C" glmrt_status_t glmrt_b200_block_norm_async(const glmrt_b200_block_norm_args_t* p, void* cuda_stream) {
  if (p == nullptr) return fail(GLMRT_STATUS_INVALID_ARGUMENT, "block_norm: null arguments");
  if (p->dtype > GLMRT_B200_DTYPE_F32 || p->weight_dtype > GLMRT_B200_DTYPE_F32)
    return fail(GLMRT_STATUS_INVALID_ARGUMENT, "block_norm: dtype must be GLMRT_B200_DTYPE_BF16 or _F32");
  if (p->width == 0 || p->width > kMaxWidth)
    return fail(GLMRT_STATUS_INVALID_ARGUMENT, "block_norm: width must be 1..32768");
  if (p->rows > 0x7fffffffu) return fail(GLMRT_STATUS_INVALID_ARGUMENT, "block_norm: too many rows");
  if (!(p->eps >= 0.0f) || !isfinite(p->eps) || !isfinite(p->scale))
    return fail(GLMRT_STATUS_INVALID_ARGUMENT, "block_norm: eps must be finite and not negative, scale finite");
  if (p->rows == 0) return ok();
  const size_t size = p->dtype == GLMRT_B200_DTYPE_BF16 ? 2 : 4, wsize = p->weight_dtype == GLMRT_B200_DTYPE_BF16 ? 2 : 4;
  const bool branch = p->delta.ptr != nullptr;
  if (!branch && (p->post_weight.ptr != nullptr || p->gate.ptr != nullptr || p->residual_out.ptr != nullptr))
    return fail(GLMRT_STATUS_INVALID_ARGUMENT, "block_norm: post_weight, gate and residual_out need a delta");
  // the widest access that the width, every address and every stride allow: 16 bytes, 8 bytes (bf16 rows) or one value
  int align = p->width % (16 / size) == 0 ? 16 : p->width % (8 / size) == 0 ? 8 : 0;
  auto aligned_to = [&](uintptr_t v) {
    while (align != 0 && v % static_cast<uintptr_t>(align) != 0) align = align == 16 ? 8 : 0;
  };
  Span spans[4];                              // residual, delta, residual_out, normalized
  auto rows_ok = [&](const glmrt_device_buffer_t& b, size_t row_stride, Span* span, const char* what) {
    if (b.ptr == nullptr) return fail(GLMRT_STATUS_INVALID_ARGUMENT, std::string("block_norm ") + what + ": null buffer");
    if (row_stride < p->width) return fail(GLMRT_STATUS_INVALID_ARGUMENT, std::string("block_norm ") + what + ": row stride below width");
    size_t need = 0;
    if (!checked_mul(p->rows - 1, row_stride, &need) || need > (SIZE_MAX >> 3) || b.bytes < (need + p->width) * size)
      return fail(GLMRT_STATUS_BUFFER_TOO_SMALL, std::string("block_norm ") + what + ": buffer too small");
    const uintptr_t at = reinterpret_cast<uintptr_t>(b.ptr);
    if (at % size != 0) return fail(GLMRT_STATUS_INVALID_ARGUMENT, std::string("block_norm ") + what + ": misaligned");
    aligned_to(at);
    if (p->rows > 1) aligned_to(row_stride * size);
    *span = Span{at, at + (need + p->width) * size, row_stride};
    return GLMRT_STATUS_OK;
  };
  GLMRT_RETURN_IF_ERROR(rows_ok(p->residual, p->residual_stride, &spans[0], "residual"));
  GLMRT_RETURN_IF_ERROR(rows_ok(p->normalized, p->normalized_stride, &spans[3], "normalized"));
  if (branch) {
    GLMRT_RETURN_IF_ERROR(rows_ok(p->delta, p->delta_stride, &spans[1], "delta"));
    GLMRT_RETURN_IF_ERROR(rows_ok(p->residual_out, p->residual_out_stride, &spans[2], "residual_out"));
    if (overlap(spans[2], spans[3]))
      return fail(GLMRT_STATUS_INVALID_ARGUMENT, "block_norm: residual_out and normalized overlap");
  }
  // an output may take the place of an input, row for row; any other overlap would be read after it was written
  for (int out : {2, 3})
    for (int in : {0, 1}) {
      if (!branch && (out == 2 || in == 1)) continue;
      if (overlap(spans[out], spans[in]) && (spans[out].lo != spans[in].lo || (spans[out].stride != spans[in].stride && p->rows > 1)))
        return fail(GLMRT_STATUS_INVALID_ARGUMENT, "block_norm: an output overlaps an input without being it");
    }
  auto weight_ok = [&](const glmrt_device_buffer_t& b, const char* what) {
    if (b.bytes < p->width * wsize) return fail(GLMRT_STATUS_BUFFER_TOO_SMALL, std::string("block_norm ") + what + ": buffer too small");
    const uintptr_t at = reinterpret_cast<uintptr_t>(b.ptr);
    if (at % wsize != 0) return fail(GLMRT_STATUS_INVALID_ARGUMENT, std::string("block_norm ") + what + ": misaligned");
    const Span s{at, at + p->width * wsize, 0};
    if (overlap(s, spans[3]) || (branch && overlap(s, spans[2])))
      return fail(GLMRT_STATUS_INVALID_ARGUMENT, std::string("block_norm ") + what + ": overlaps an output");
    // (the narrower pieces are four values: 8 bytes of bf16 weights, 16 of float32)
    if (wsize == 4 && at % 16 != 0) align = 0;
    else aligned_to(at);
    return GLMRT_STATUS_OK;
  };
  if (p->norm_weight.ptr == nullptr) return fail(GLMRT_STATUS_INVALID_ARGUMENT, "block_norm norm_weight: null buffer");
  GLMRT_RETURN_IF_ERROR(weight_ok(p->norm_weight, "norm_weight"));
  if (p->post_weight.ptr != nullptr) GLMRT_RETURN_IF_ERROR(weight_ok(p->post_weight, "post_weight"));
  if (p->gate.ptr != nullptr) {
    if (p->gate_col_stride > 1) return fail(GLMRT_STATUS_INVALID_ARGUMENT, "block_norm gate: column stride must be 0 or 1");
    size_t need = 0;
    if (!checked_mul(p->rows - 1, p->gate_row_stride, &need) || need > (SIZE_MAX >> 3) ||
        p->gate.bytes < (need + (p->gate_col_stride ? p->width : 1)) * size)
      return fail(GLMRT_STATUS_BUFFER_TOO_SMALL, "block_norm gate: buffer too small");
    const uintptr_t at = reinterpret_cast<uintptr_t>(p->gate.ptr);
    if (at % size != 0) return fail(GLMRT_STATUS_INVALID_ARGUMENT, "block_norm gate: misaligned");
    const Span s{at, at + (need + (p->gate_col_stride ? p->width : 1)) * size, 0};
    if (overlap(s, spans[2]) || overlap(s, spans[3]))
      return fail(GLMRT_STATUS_INVALID_ARGUMENT, "block_norm gate: overlaps an output");
    if (p->gate_col_stride != 0) {
      aligned_to(at);
      aligned_to(p->gate_row_stride * size);
    }
  }
  GLMRT_RETURN_IF_ERROR(require_cuda());
  NormArgs a{};
  a.residual = p->residual.ptr; a.delta = p->delta.ptr; a.norm_w = p->norm_weight.ptr; a.post_w = p->post_weight.ptr;
  a.gate = p->gate.ptr; a.residual_out = p->residual_out.ptr; a.normalized = p->normalized.ptr;
  a.residual_stride = p->residual_stride; a.delta_stride = p->delta_stride; a.gate_rs = p->gate_row_stride;
  a.gate_cs = p->gate_col_stride; a.residual_out_stride = p->residual_out_stride; a.normalized_stride = p->normalized_stride;
  a.rows = static_cast<int>(p->rows); a.width = static_cast<int>(p->width);
  a.scale = p->scale; a.eps = p->eps;
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  GLMRT_RETURN_IF_ERROR(size == 2 ? (wsize == 2 ? dispatch_vec<uint16_t, uint16_t>(a, align, s) : dispatch_vec<uint16_t, float>(a, align, s))
                                  : (wsize == 2 ? dispatch_vec<float, uint16_t>(a, align, s) : dispatch_vec<float, float>(a, align, s)));
  GLMRT_LAUNCH_CHECK("block_norm_kernel");
  return ok();
}
