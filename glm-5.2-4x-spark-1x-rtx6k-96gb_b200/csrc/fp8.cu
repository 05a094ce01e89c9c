// Products in 8-bit floating point with a scale for each block of 128: the dense projections beside
// the routed experts (the shared expert of a sparse layer is their user, shared_expert.py).
//
//   activations  E4M3, one scale per row and 128 columns: the smallest power of two with
//                amax / scale <= 448, so that dividing by it is exact and the codes do not depend on
//                how a quotient is rounded
//   weights      E4M3 [n, k] and one float32 scale per 128 x 128 block
//   product      y[m, n] = sum over blocks b of sx[m, b] sw[n / 128, b] sum over k in b of q[m, k] w[n, k],
//                float32 sums
#include <initializer_list>

#include "common.cuh"
#include "fp8.cuh"
#include "internal.h"

namespace glmrt {
namespace {

constexpr int kBlock = kFp8Block;

// Eight lanes per (row, 128-column block), sixteen values a lane (two 16-byte loads of bf16 in flight, one 16-byte store
// of codes); a CTA takes eight rows of four neighbouring blocks, so that the scales leave as whole sectors.  Bound by
// memory (3 bytes a bf16 value, 5 a float32 one): 8192 x 6144 bf16 25 us = 6.0 TB/s, float32 38 us = 6.6 TB/s (bf16 with eight
// values a lane, and blocks of one row next to each other in a CTA, 33 us).  kVec: the rows' pieces of eight values are 16-byte aligned.
constexpr int kQuantBlocks = 4, kQuantRows = 256 / 8 / kQuantBlocks;       // of a CTA
template <typename T, bool kVec>
__global__ void __launch_bounds__(256) fp8_quantize_rows_kernel(const T* __restrict__ in, size_t stride, uint8_t* __restrict__ codes,
                                                                float* __restrict__ scales, int rows, int cols, int scale_stride) {
  pdl_wait();
  pdl_launch_dependents();      // after the wait: a successor may then rely on everything before this kernel
  const uint32_t blocks = (cols + kBlock - 1) / kBlock, tiles = (blocks + kQuantBlocks - 1) / kQuantBlocks;
  const uint32_t sub = threadIdx.x % 8, group = threadIdx.x / 8, row_tile = blockIdx.x / tiles;
  const uint32_t row = row_tile * kQuantRows + group / kQuantBlocks, b = (blockIdx.x - row_tile * tiles) * kQuantBlocks + group % kQuantBlocks;
  const uint32_t c = b * kBlock + sub * 16;
  const bool in_rows = row < static_cast<uint32_t>(rows), has_values = in_rows && c < static_cast<uint32_t>(cols);   // cols % 16 == 0
  float v[16] = {};
  if (has_values) {
    const T* src = in + row * stride + c;
    if constexpr (kVec) {
      alignas(16) T t[16];
#pragma unroll
      for (int i = 0; i < 16; i += 16 / static_cast<int>(sizeof(T))) *reinterpret_cast<uint4*>(t + i) = *reinterpret_cast<const uint4*>(src + i);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = fp8_input(t[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = fp8_input(src[i]);
    }
  }
  uint32_t amax = 0u;
#pragma unroll
  for (int i = 0; i < 16; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  float inv;
  const float scale = fp8_block_scale(amax, &inv);
  if (has_values) {
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = fp8_pack4(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv, v[4 * i + 3] * inv);
    *reinterpret_cast<uint4*>(codes + static_cast<size_t>(row) * cols + c) = make_uint4(q[0], q[1], q[2], q[3]);
  }
  if (sub == 0 && in_rows && b < blocks) scales[static_cast<size_t>(b) * scale_stride + row] = scale;
}

size_t round256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }
size_t blocks_of(size_t k) { return (k + kBlock - 1) / kBlock; }
size_t padded(size_t rows) { return (rows + 255) & ~static_cast<size_t>(255); }   // whole tiles of the products
size_t rows_bytes(size_t rows, size_t k) { return round256(rows * k) + padded(rows) * blocks_of(k) * 4; }

glmrt_status_t check_dims(size_t rows, size_t n, size_t k, const char* what) {
  if (n == 0 || k == 0 || k % 16 != 0)
    return fail(GLMRT_STATUS_INVALID_ARGUMENT, std::string(what) + ": sizes must be positive and the summed one a multiple of 16");
  if (rows > (1u << 24) || n > (1u << 24) || k > (1u << 24))
    return fail(GLMRT_STATUS_INVALID_ARGUMENT, std::string(what) + ": sizes must be at most 2^24");
  return GLMRT_STATUS_OK;
}
glmrt_status_t check_buffer(const glmrt_device_buffer_t& b, size_t need, size_t align, const char* what) {
  if (b.ptr == nullptr) return fail(GLMRT_STATUS_INVALID_ARGUMENT, std::string(what) + ": null buffer");
  if (b.bytes < need) return fail(GLMRT_STATUS_BUFFER_TOO_SMALL, std::string(what) + ": buffer too small");
  if (reinterpret_cast<uintptr_t>(b.ptr) % align != 0)
    return fail(GLMRT_STATUS_INVALID_ARGUMENT, std::string(what) + ": misaligned buffer");
  return GLMRT_STATUS_OK;
}

// What a call writes (its first `need` bytes) must lie apart from everything it reads and from its workspace: tiles of
// the output are written while others still read the rows.
struct Span { const void* ptr; size_t bytes; };
glmrt_status_t check_apart(const Span& out, std::initializer_list<Span> others, const char* what) {
  const uintptr_t o = reinterpret_cast<uintptr_t>(out.ptr);
  for (const Span& s : others) {
    const uintptr_t i = reinterpret_cast<uintptr_t>(s.ptr);
    if (i < o + out.bytes && o < i + s.bytes) return fail(GLMRT_STATUS_INVALID_ARGUMENT, std::string(what) + ": overlaps another buffer of the call");
  }
  return GLMRT_STATUS_OK;
}

glmrt_status_t launch_quantize(const void* in, uint32_t dtype, size_t stride, uint8_t* codes, float* scales, size_t rows,
                               size_t cols, size_t scale_stride, cudaStream_t s) {
  const size_t size = dtype == GLMRT_B200_DTYPE_BF16 ? 2 : 4;
  const size_t ctas = (rows + kQuantRows - 1) / kQuantRows * ((blocks_of(cols) + kQuantBlocks - 1) / kQuantBlocks);
  const bool vec = reinterpret_cast<uintptr_t>(in) % 16 == 0 && stride * size % 16 == 0;
  const dim3 grid(static_cast<unsigned>(ctas)), block(256);
  const int m = static_cast<int>(rows), n = static_cast<int>(cols), ss = static_cast<int>(scale_stride);
  auto run = [&](auto kernel, auto* src) { launch_pdl(kernel, grid, block, 0, s, src, stride, codes, scales, m, n, ss); };
  const auto* bf = static_cast<const uint16_t*>(in);
  const auto* f = static_cast<const float*>(in);
  if (size == 2) vec ? run(fp8_quantize_rows_kernel<uint16_t, true>, bf) : run(fp8_quantize_rows_kernel<uint16_t, false>, bf);
  else vec ? run(fp8_quantize_rows_kernel<float, true>, f) : run(fp8_quantize_rows_kernel<float, false>, f);
  GLMRT_LAUNCH_CHECK("fp8_quantize_rows_kernel");
  return GLMRT_STATUS_OK;
}

}  // namespace
}  // namespace glmrt

using namespace glmrt;

extern "C" glmrt_status_t glmrt_b200_fp8_quantize_rows_async(const glmrt_b200_fp8_quantize_rows_args_t* args, void* cuda_stream) {
  if (args == nullptr) return fail(GLMRT_STATUS_INVALID_ARGUMENT, "fp8_quantize_rows: null arguments");
  const auto& [input, codes, scales, rows, cols, input_row_stride, dtype] = *args;
  GLMRT_RETURN_IF_ERROR(check_dims(rows, 1, cols, "fp8_quantize_rows"));
  if (dtype > GLMRT_B200_DTYPE_F32 || input_row_stride < cols || input_row_stride > (size_t{1} << 32))
    return fail(GLMRT_STATUS_INVALID_ARGUMENT, "fp8_quantize_rows: unknown dtype, or row stride below cols");
  if (rows == 0) return ok();
  const size_t size = dtype == GLMRT_B200_DTYPE_BF16 ? 2 : 4;
  GLMRT_RETURN_IF_ERROR(check_buffer(input, ((rows - 1) * input_row_stride + cols) * size, size, "fp8_quantize_rows input"));
  GLMRT_RETURN_IF_ERROR(check_buffer(codes, rows * cols, 16, "fp8_quantize_rows codes"));
  GLMRT_RETURN_IF_ERROR(check_buffer(scales, rows * blocks_of(cols) * 4, 4, "fp8_quantize_rows scales"));
  const Span in{input.ptr, ((rows - 1) * input_row_stride + cols) * size}, sc{scales.ptr, rows * blocks_of(cols) * 4};
  GLMRT_RETURN_IF_ERROR(check_apart({codes.ptr, rows * cols}, {in, sc}, "fp8_quantize_rows codes"));
  GLMRT_RETURN_IF_ERROR(check_apart(sc, {in}, "fp8_quantize_rows scales"));
  GLMRT_RETURN_IF_ERROR(require_cuda());
  GLMRT_RETURN_IF_ERROR(launch_quantize(input.ptr, dtype, input_row_stride, static_cast<uint8_t*>(codes.ptr),
                                        static_cast<float*>(scales.ptr), rows, cols, rows, static_cast<cudaStream_t>(cuda_stream)));
  return ok();
}

extern "C" glmrt_status_t glmrt_b200_fp8_block_linear_workspace(size_t rows, size_t n, size_t k, size_t* out_bytes) {
  if (out_bytes == nullptr) return fail(GLMRT_STATUS_INVALID_ARGUMENT, "fp8_block_linear_workspace: null output");
  GLMRT_RETURN_IF_ERROR(check_dims(rows, n, k, "fp8_block_linear"));
  *out_bytes = rows <= kFp8OwnRows ? 0 : rows_bytes(rows, k);
  return ok();
}

extern "C" glmrt_status_t glmrt_b200_fp8_block_linear_async(const glmrt_b200_fp8_block_linear_args_t* args, void* cuda_stream) {
  if (args == nullptr) return fail(GLMRT_STATUS_INVALID_ARGUMENT, "fp8_block_linear: null arguments");
  const auto& [x_bf16, weight_codes, weight_scales, output, workspace, rows, n, k, x_row_stride, out_dtype] = *args;
  GLMRT_RETURN_IF_ERROR(check_dims(rows, n, k, "fp8_block_linear"));
  if (out_dtype > GLMRT_B200_DTYPE_F32 || x_row_stride < k || x_row_stride > (size_t{1} << 32))
    return fail(GLMRT_STATUS_INVALID_ARGUMENT, "fp8_block_linear: unknown output dtype, or x row stride below k");
  if (rows == 0) return ok();
  const size_t osize = out_dtype == GLMRT_B200_DTYPE_BF16 ? 2 : 4;
  GLMRT_RETURN_IF_ERROR(check_buffer(x_bf16, ((rows - 1) * x_row_stride + k) * 2, 2, "fp8_block_linear x"));
  GLMRT_RETURN_IF_ERROR(check_buffer(weight_codes, n * k, 16, "fp8_block_linear weight_codes"));
  GLMRT_RETURN_IF_ERROR(check_buffer(weight_scales, blocks_of(n) * blocks_of(k) * 4, 4, "fp8_block_linear weight_scales"));
  GLMRT_RETURN_IF_ERROR(check_buffer(output, rows * n * osize, osize, "fp8_block_linear output"));
  const bool own = rows <= kFp8OwnRows;      // the product quantises so few rows itself
  if (!own) GLMRT_RETURN_IF_ERROR(check_buffer(workspace, rows_bytes(rows, k), 256, "fp8_block_linear workspace"));
  const Span x{x_bf16.ptr, ((rows - 1) * x_row_stride + k) * 2}, wc{weight_codes.ptr, n * k}, wsc{weight_scales.ptr, blocks_of(n) * blocks_of(k) * 4},
      out{output.ptr, rows * n * osize};
  GLMRT_RETURN_IF_ERROR(check_apart(out, {x, wc, wsc}, "fp8_block_linear output"));
  if (!own) GLMRT_RETURN_IF_ERROR(check_apart({workspace.ptr, rows_bytes(rows, k)}, {x, wc, wsc, out}, "fp8_block_linear workspace"));
  GLMRT_RETURN_IF_ERROR(require_cuda());
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  uint8_t* codes = static_cast<uint8_t*>(workspace.ptr);
  float* scales = reinterpret_cast<float*>(codes + round256(rows * k));
  if (!own) GLMRT_RETURN_IF_ERROR(launch_quantize(x_bf16.ptr, GLMRT_B200_DTYPE_BF16, x_row_stride, codes, scales, rows, k, padded(rows), s));
  Fp8Gemm g{codes, scales, static_cast<const uint8_t*>(weight_codes.ptr), nullptr, static_cast<const float*>(weight_scales.ptr),
            nullptr, output.ptr, nullptr, static_cast<int>(rows), static_cast<int>(n), static_cast<int>(k),
            static_cast<int>(padded(rows)), 0, own ? static_cast<const uint16_t*>(x_bf16.ptr) : nullptr, x_row_stride};
  GLMRT_RETURN_IF_ERROR(launch_fp8_gemm(g, out_dtype == GLMRT_B200_DTYPE_BF16 ? 0 : 1, s));
  return ok();
}

extern "C" glmrt_status_t glmrt_b200_fp8_gated_mlp_workspace(size_t rows, size_t hidden, size_t inter, size_t* out_bytes) {
  if (out_bytes == nullptr) return fail(GLMRT_STATUS_INVALID_ARGUMENT, "fp8_gated_mlp_workspace: null output");
  GLMRT_RETURN_IF_ERROR(check_dims(rows, inter, hidden, "fp8_gated_mlp"));
  GLMRT_RETURN_IF_ERROR(check_dims(rows, hidden, inter, "fp8_gated_mlp"));
  *out_bytes = (rows <= kFp8OwnRows ? 0 : rows_bytes(rows, hidden)) + rows_bytes(rows, inter);
  return ok();
}

extern "C" glmrt_status_t glmrt_b200_fp8_gated_mlp_async(const glmrt_b200_fp8_gated_mlp_args_t* args, void* cuda_stream) {
  if (args == nullptr) return fail(GLMRT_STATUS_INVALID_ARGUMENT, "fp8_gated_mlp: null arguments");
  const auto& [x_bf16, gate_codes, gate_scales, up_codes, up_scales, down_codes, down_scales, output_bf16, workspace, rows,
               hidden, inter, x_row_stride] = *args;
  size_t need = 0;
  GLMRT_RETURN_IF_ERROR(glmrt_b200_fp8_gated_mlp_workspace(rows, hidden, inter, &need));
  if (x_row_stride < hidden || x_row_stride > (size_t{1} << 32))
    return fail(GLMRT_STATUS_INVALID_ARGUMENT, "fp8_gated_mlp: x row stride below hidden");
  if (rows == 0) return ok();
  const size_t scale_bytes = blocks_of(hidden) * blocks_of(inter) * 4;
  GLMRT_RETURN_IF_ERROR(check_buffer(x_bf16, ((rows - 1) * x_row_stride + hidden) * 2, 2, "fp8_gated_mlp x"));
  GLMRT_RETURN_IF_ERROR(check_buffer(gate_codes, hidden * inter, 16, "fp8_gated_mlp gate_codes"));
  GLMRT_RETURN_IF_ERROR(check_buffer(up_codes, hidden * inter, 16, "fp8_gated_mlp up_codes"));
  GLMRT_RETURN_IF_ERROR(check_buffer(down_codes, hidden * inter, 16, "fp8_gated_mlp down_codes"));
  GLMRT_RETURN_IF_ERROR(check_buffer(gate_scales, scale_bytes, 4, "fp8_gated_mlp gate_scales"));
  GLMRT_RETURN_IF_ERROR(check_buffer(up_scales, scale_bytes, 4, "fp8_gated_mlp up_scales"));
  GLMRT_RETURN_IF_ERROR(check_buffer(down_scales, scale_bytes, 4, "fp8_gated_mlp down_scales"));
  GLMRT_RETURN_IF_ERROR(check_buffer(output_bf16, rows * hidden * 2, 2, "fp8_gated_mlp output"));
  GLMRT_RETURN_IF_ERROR(check_buffer(workspace, need, 256, "fp8_gated_mlp workspace"));
  const Span x{x_bf16.ptr, ((rows - 1) * x_row_stride + hidden) * 2}, gc{gate_codes.ptr, hidden * inter}, gs{gate_scales.ptr, scale_bytes},
      uc{up_codes.ptr, hidden * inter}, us{up_scales.ptr, scale_bytes}, dc{down_codes.ptr, hidden * inter}, ds{down_scales.ptr, scale_bytes},
      out{output_bf16.ptr, rows * hidden * 2};
  // (the rows have been read when the last product starts, so the output may take their place where they are whole)
  GLMRT_RETURN_IF_ERROR(check_apart(out, {gc, gs, uc, us, dc, ds}, "fp8_gated_mlp output"));
  GLMRT_RETURN_IF_ERROR(check_apart({workspace.ptr, need}, {x, gc, gs, uc, us, dc, ds, out}, "fp8_gated_mlp workspace"));
  GLMRT_RETURN_IF_ERROR(require_cuda());
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  uint8_t* xq = static_cast<uint8_t*>(workspace.ptr);
  float* xs = reinterpret_cast<float*>(xq + round256(rows * hidden));
  uint8_t* aq = rows <= kFp8OwnRows ? xq : xq + rows_bytes(rows, hidden);
  float* as = reinterpret_cast<float*>(aq + round256(rows * inter));
  const bool own = rows <= kFp8OwnRows;      // the product quantises so few rows itself
  if (!own) GLMRT_RETURN_IF_ERROR(launch_quantize(x_bf16.ptr, GLMRT_B200_DTYPE_BF16, x_row_stride, xq, xs, rows, hidden, padded(rows), s));
  const int m = static_cast<int>(rows), h = static_cast<int>(hidden), i = static_cast<int>(inter), pad = static_cast<int>(padded(rows));
  const Fp8Gemm up{xq, xs, static_cast<const uint8_t*>(gate_codes.ptr), static_cast<const uint8_t*>(up_codes.ptr),
                   static_cast<const float*>(gate_scales.ptr), static_cast<const float*>(up_scales.ptr), aq, as, m, i, h, pad, pad,
                   own ? static_cast<const uint16_t*>(x_bf16.ptr) : nullptr, x_row_stride};
  const Fp8Gemm down{aq, as, static_cast<const uint8_t*>(down_codes.ptr), nullptr, static_cast<const float*>(down_scales.ptr),
                     nullptr, output_bf16.ptr, nullptr, m, h, i, pad, 0};
  GLMRT_RETURN_IF_ERROR(launch_fp8_gemm(up, 2, s));
  GLMRT_RETURN_IF_ERROR(launch_fp8_gemm(down, 0, s));
  return ok();
}
