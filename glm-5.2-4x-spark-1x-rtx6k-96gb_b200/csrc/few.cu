// A whole sparse layer for a few tokens (at most kFewMaxRows rows): router, experts on bf16
// activations (W4A16, the arithmetic of the reference's decode kernels: native/cuda/kernels/
// b12x_direct.cu:171-201,989-1541), weighted combine, and the residual and shared rows added on top.
//
//   act[r]  = weight[r] * silu(gate x) * (up x)          r = (token, slot), float32
//   out[t]  = residual[t] + (shared[t] + sum over slots down act[t, slot])
//
// with W = E2M1 code * E4M3 block scale * scale_2.  Nothing is rounded between the bf16 rows and the
// bf16 result except where a comment says so.
#include "common.cuh"
#include "internal.h"

namespace glmrt {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
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

glmrt_status_t launch_few_simt(const FewArgs& a, cudaStream_t s) {
  launch_pdl(few_fc1_simt_kernel, dim3((a.inter + 7) / 8, a.rows * a.top_k), dim3(256), 0, s, a);
  GLMRT_LAUNCH_CHECK("few_fc1_simt_kernel");
  launch_pdl(few_fc2_simt_kernel, dim3((a.hidden + 7) / 8, a.rows), dim3(256), 0, s, a);
  GLMRT_LAUNCH_CHECK("few_fc2_simt_kernel");
  return GLMRT_STATUS_OK;
}

}  // namespace glmrt
