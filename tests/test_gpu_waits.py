"""GPU test of a bounded wait that runs out: every lane of the warp gets the same answer."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

pytestmark = pytest.mark.gpu

# One warp whose lower half waits for a phase that is complete and whose upper half waits for one that nothing
# completes (then for the first as well): the wait ends by its own limit, and both halves are told so.
SOURCE = r"""
#include <atomic>
#include "common.cuh"
#include "internal.h"
#include "tc_ptx.cuh"
__global__ void waits(uint32_t* out) {
  __shared__ uint64_t bars[2];
  __shared__ uint32_t abort_word;
  if (threadIdx.x == 0) {
    abort_word = 0u;
    glmrt::tc::mbar_init(&bars[0], 1);
    glmrt::tc::mbar_init(&bars[1], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    glmrt::tc::mbar_arrive(&bars[0]);
  }
  __syncwarp();
  out[threadIdx.x] = glmrt::tc::mbar_wait_hot(&bars[0], 0u, &abort_word);
  out[32 + threadIdx.x] = *static_cast<volatile uint32_t*>(&abort_word);
  __syncwarp();
  out[64 + threadIdx.x] = glmrt::tc::mbar_wait_hot(&bars[threadIdx.x / 16], 0u, &abort_word);
  out[96 + threadIdx.x] = *static_cast<volatile uint32_t*>(&abort_word);
}
extern "C" int run(uint32_t* out, cudaStream_t stream) {
  waits<<<1, 32, 0, stream>>>(out);
  return static_cast<int>(cudaGetLastError());
}
"""


def test_expired_wait_has_one_answer_for_the_warp(pkg, tmp_path):
    csrc = os.path.join(os.path.dirname(pkg.__file__), "csrc")
    (tmp_path / "waits.cu").write_text(SOURCE)
    lib = tmp_path / "libwaits.so"
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    subprocess.run([nvcc, "-std=c++17", "-O3", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr", "-shared",
                    "-Xcompiler", "-fPIC", "-I", csrc, "-I", os.path.join(csrc, "..", "..", "include"), "-o", str(lib), str(tmp_path / "waits.cu")],
                   check=True, timeout=300)
    out = torch.full((4, 32), 9, dtype=torch.int32, device="cuda")
    assert C.CDLL(str(lib)).run(C.c_void_p(out.data_ptr()), C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()
    assert out.float().mean(1).tolist() == [1.0, 0.0, 0.0, 1.0]
