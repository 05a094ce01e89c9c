"""Dense products in 8-bit floating point with a scale for each block of 128 (csrc/fp8.cu).

Weights: E4M3 ``[n, k]`` with one float32 scale per 128 x 128 block, ``[ceil(n/128), ceil(k/128)]``.
Activations: bf16 rows, quantised in the call with one power-of-two scale per row and 128 columns
(the smallest with ``amax / scale <= 448``).  Sums are float32.  ``k`` is a multiple of 16; rows, ``n``
and the last block may be ragged.  A row with a NaN or an infinity gives NaN outputs in that row only.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct

import torch

from . import launch
from . import native as N

BLOCK = 128
E4M3 = torch.float8_e4m3fn
_CODE_TYPES = (E4M3, torch.uint8)
_ROW_TYPES = (torch.bfloat16,)
_QUANT_ARGS = struct.Struct("@" + launch.BUFFER * 3 + "3QI4x")       # glmrt_b200_fp8_quantize_rows_args_t
_LINEAR_ARGS = struct.Struct("@" + launch.BUFFER * 5 + "4QI4x")      # glmrt_b200_fp8_block_linear_args_t
_MLP_ARGS = struct.Struct("@" + launch.BUFFER * 9 + "4Q")            # glmrt_b200_fp8_gated_mlp_args_t


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _rows(x: torch.Tensor, k: int, types: tuple, what: str) -> tuple[int, tuple, int]:
    """Number, packed buffer and row stride of the rows."""
    if x.dim() != 2 or x.shape[1] != k or x.dtype not in types:
        raise ValueError(f"{what} must be [rows, {k}] of type {' or '.join(str(t) for t in types)}")
    if not x.is_cuda:
        raise ValueError(f"{what} must be on a CUDA device")
    rows = x.shape[0]
    buf, stride = launch.rows_buffer(x, rows, k, x.itemsize, what)
    return rows, buf, stride


def _weight(codes: torch.Tensor, scales: torch.Tensor, n: int, k: int, index: int, what: str) -> tuple:
    """Packed buffers of a weight's codes and scales."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    if codes.shape != (n, k) or codes.dtype not in _CODE_TYPES or not codes.is_contiguous():
        raise ValueError(f"{what} codes must be a contiguous E4M3 (or uint8) tensor [{n}, {k}]")
    if scales.shape != (nb, kb) or scales.dtype is not torch.float32 or not scales.is_contiguous():
        raise ValueError(f"{what} scales must be a contiguous float32 tensor [{nb}, {kb}]")
    if codes.get_device() != index or scales.get_device() != index:
        raise ValueError(f"{what} must be on the device of the rows")
    return codes.data_ptr(), n * k, 0, 0, scales.data_ptr(), nb * kb * 4, 0, 0


def quantize_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales (amax / 448 per 128 x 128 block) of a weight; done once at load."""
    n, k = weight.shape
    pad = torch.nn.functional.pad(weight.float(), (0, -k % BLOCK, 0, -n % BLOCK))
    b = pad.view(_blocks(n), BLOCK, _blocks(k), BLOCK)
    scales = b.abs().amax(dim=(1, 3)) / 448.0
    scales = torch.where(scales > 0, scales, torch.ones_like(scales))       # of zeros, or so small that the quotient is zero
    codes = (b / scales[:, None, :, None]).reshape(pad.shape)[:n, :k].clamp(-448, 448).to(E4M3)
    return codes.contiguous(), scales


def quantize_rows(x: torch.Tensor, lib: N.NativeLibrary | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows' codes ``[rows, k]`` (E4M3) and scales ``[ceil(k/128), rows]``; x bf16 or float32."""
    k = x.shape[1] if x.dim() == 2 else 0
    rows, buf, stride = _rows(x, k, (torch.bfloat16, torch.float32), "quantize_rows: x")
    codes = torch.empty((rows, k), dtype=E4M3, device=x.device)
    scales = torch.empty((_blocks(k), rows), dtype=torch.float32, device=x.device)
    launch.call(lib, "glmrt_b200_fp8_quantize_rows_async",
                _QUANT_ARGS.pack(*buf, *launch.buffer(codes), *launch.buffer(scales), rows, k, stride,
                                 N.DTYPE_BF16 if x.dtype == torch.bfloat16 else N.DTYPE_F32), x.get_device())
    return codes, scales


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(lib: N.NativeLibrary, symbol: str, *sizes: int) -> int:
    need = C.c_size_t(0)
    lib.call(symbol, *[C.c_size_t(v) for v in sizes], C.byref(need))
    return need.value


def _output(out: torch.Tensor | None, rows: int, n: int, dtype: torch.dtype, x: torch.Tensor) -> torch.Tensor:
    if out is None:
        return x.new_empty((rows, n)) if dtype is x.dtype else x.new_empty((rows, n), dtype=dtype)
    if out.shape != (rows, n) or out.dtype is not dtype or out.get_device() != x.get_device() or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {dtype} tensor [{rows}, {n}] on the rows' device")
    return out


def _workspace(lib: N.NativeLibrary, symbol: str, x: torch.Tensor, *sizes: int) -> torch.Tensor | None:
    need = _workspace_bytes(lib, symbol, *sizes)
    return x.new_empty((need + 1) // 2) if need else None                     # of bf16 rows: two bytes each


def block_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, out: torch.Tensor | None = None,
                 out_dtype: torch.dtype = torch.bfloat16, lib: N.NativeLibrary | None = None) -> torch.Tensor:
    """``x @ weight.T`` of bf16 rows and an E4M3 weight ``[n, k]``; out bf16 or float32."""
    lib = lib or N.library()
    if codes.dim() != 2:
        raise ValueError("block_linear: codes must be [n, k]")
    n, k = codes.shape
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("block_linear: out_dtype must be bfloat16 or float32")
    rows, buf, stride = _rows(x, k, _ROW_TYPES, "block_linear: x")
    index = x.get_device()
    weight = _weight(codes, scales, n, k, index, "block_linear: weight")
    out = _output(out, rows, n, out_dtype, x)
    ws = _workspace(lib, "glmrt_b200_fp8_block_linear_workspace", x, rows, n, k)
    launch.call(lib, "glmrt_b200_fp8_block_linear_async",
                _LINEAR_ARGS.pack(*buf, *weight, *launch.buffer(out), *launch.buffer(ws),
                                  rows, n, k, stride, N.DTYPE_BF16 if out_dtype is torch.bfloat16 else N.DTYPE_F32), index)
    return out


def gated_mlp(x: torch.Tensor, gate_codes: torch.Tensor, gate_scales: torch.Tensor, up_codes: torch.Tensor,
              up_scales: torch.Tensor, down_codes: torch.Tensor, down_scales: torch.Tensor,
              out: torch.Tensor | None = None, lib: N.NativeLibrary | None = None) -> torch.Tensor:
    """``down(silu(gate(x)) * up(x))`` with gate / up ``[inter, hidden]`` and down ``[hidden, inter]``; the
    activation between the products stays float32 until it is quantised like the rows."""
    lib = lib or N.library()
    if gate_codes.dim() != 2:
        raise ValueError("gated_mlp: gate codes must be [inter, hidden]")
    inter, hidden = gate_codes.shape
    rows, buf, stride = _rows(x, hidden, _ROW_TYPES, "gated_mlp: x")
    index = x.get_device()
    gate = _weight(gate_codes, gate_scales, inter, hidden, index, "gated_mlp: gate")
    up = _weight(up_codes, up_scales, inter, hidden, index, "gated_mlp: up")
    down = _weight(down_codes, down_scales, hidden, inter, index, "gated_mlp: down")
    out = _output(out, rows, hidden, torch.bfloat16, x)
    ws = _workspace(lib, "glmrt_b200_fp8_gated_mlp_workspace", x, rows, hidden, inter)
    launch.call(lib, "glmrt_b200_fp8_gated_mlp_async",
                _MLP_ARGS.pack(*buf, *gate, *up, *down, *launch.buffer(out), *launch.buffer(ws), rows, hidden, inter, stride), index)
    return out
