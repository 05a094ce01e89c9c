// Number formats and the activation quantiser's block arithmetic of the 8-bit products (fp8.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace glmrt {

constexpr int kFp8Block = 128;   // columns per activation scale, rows and columns per weight scale

// One product of quantised rows x [rows, k] (E4M3, scales [ceil(k / 128)][xs_stride], xs_stride whole tiles of
// 256) with weights [n, k] (scales ws [ceil(n / 128)][ceil(k / 128)]).
// mode 0: out bf16 [rows, n]; 1: float32; 2: silu(w0 x) * (w1 x) quantised: codes [rows, n], scales
// out_scales [ceil(n / 128)][out_stride].
// x_bf16: instead of x and xs, at most kFp8OwnRows rows of bf16 that the product quantises itself.
// (Measured from a graph, against a quantiser before the product, 1 to 8 rows: n = 4096, k = 6144 6.8 / 8.2, 7.5 / 8.2,
// 8.0 / 8.2, 8.4 / 8.3, 8.8 / 8.3, 9.3 / 8.3, 9.8 / 8.3, 10.2 / 8.2 us; n = 6144, k = 2048 5.3 / 6.8, 5.3 / 6.8, 5.8 / 6.8,
// 6.0 / 6.9, 6.4 / 6.9, 6.6 / 6.9, 7.0 / 7.0, 7.0 / 6.8.  At four rows it loses 2 % there and wins 14 % here.)
constexpr size_t kFp8OwnRows = 4;
struct Fp8Gemm {
  const uint8_t* x;
  const float* xs;
  const uint8_t *w0, *w1;
  const float *ws0, *ws1;
  void* out;
  float* out_scales;
  int rows, n, k, xs_stride, out_stride;
  const uint16_t* x_bf16 = nullptr;
  size_t x_stride = 0;
};
glmrt_status_t launch_fp8_gemm(const Fp8Gemm& g, int mode, cudaStream_t stream);

#ifdef __CUDACC__
__device__ __forceinline__ float fp8_input(uint16_t v) { return bf16_bits_to_f32(v); }
__device__ __forceinline__ float fp8_input(float v) { return v; }
__device__ __forceinline__ void fp8_store(uint16_t* p, float v) { *p = f32_to_bf16_rne(v); }
__device__ __forceinline__ void fp8_store(float* p, float v) { *p = v; }

// Scale of a block whose largest magnitude has the bits `amax`: the smallest power of two with
// amax / scale <= 448 = 1.75 * 2^8, so one exponent comparison decides it.  Blocks below 2^-100 are
// scaled as if they reached it (their codes are then zero or tiny); a block with an infinity or a NaN gets
// the scale NaN, which makes every output of its row NaN.
__device__ __forceinline__ float fp8_block_scale(uint32_t amax, float* inv) {
  if (amax >= 0x7f800000u) {
    *inv = 0.0f;
    return __uint_as_float(0x7fc00000u);
  }
  amax = max(amax, (127u - 100u) << 23);
  const int e = static_cast<int>(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);   // -108 .. 120
  *inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}
// Four values to E4M3, nearest even (the inputs are at most 448 in magnitude).
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);       // one conversion for both
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float fp8_swiglu(float g, float u) {
  // fast exponential and division: a few units in the last place, against codes of four bits
  return __fdividef(g, 1.0f + __expf(-g)) * u;
}
#endif

}  // namespace glmrt
