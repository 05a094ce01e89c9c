"""Residual add and RMSNorms at the boundary of a block, in one kernel (csrc/norm.cu).

The routed layer takes rows that are already normalised; this makes them, together with the new
residual stream (python/reference/glmrt_reference/glm_moe_dsa_layer_ref.py:157-206):

    d = delta;  d *= rsqrt(mean(d^2) + eps) * post_weight;  d *= gate        (each where given)
    r = residual + scale * d
    y = r * rsqrt(mean(r^2) + eps) * norm_weight
"""
from __future__ import annotations

import struct

import torch

from . import launch
from . import native as N

_DTYPES = {torch.bfloat16: N.DTYPE_BF16, torch.float32: N.DTYPE_F32}
_ARGS = struct.Struct("@" + launch.BUFFER * 7 + "8Q2I2f")      # glmrt_b200_block_norm_args_t


_SIZES = {torch.bfloat16: 2, torch.float32: 4}


def _rows(t: torch.Tensor, shape, dtype: torch.dtype, index: int, what: str) -> tuple[tuple, int]:
    """Packed buffer and row stride of a [rows, width] tensor whose rows are contiguous inside."""
    if t.shape != shape or t.dtype is not dtype or t.get_device() != index:
        raise ValueError(f"block_norm: {what} must have the shape, type and device of residual")
    return launch.rows_buffer(t, shape[0], shape[1], _SIZES[dtype], "block_norm: " + what)


def _weight(w: torch.Tensor, width: int, index: int, what: str) -> tuple:
    if w.shape != (width,) or w.get_device() != index or not w.is_contiguous():
        raise ValueError(f"block_norm: {what} must be a contiguous [{width}] tensor on the rows' device")
    return w.data_ptr(), w.nbytes, 0, 0


def block_norm(residual: torch.Tensor, delta: torch.Tensor | None = None, *, norm_weight: torch.Tensor,
               post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
               eps: float = 1e-5, residual_out: torch.Tensor | None = None, normalized: torch.Tensor | None = None,
               lib: N.NativeLibrary | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(residual + scale * branch, its RMSNorm)``; rows bf16 or float32, weights bf16 or float32.

    ``gate``: [rows, 1], [1, width] or [rows, width] of the rows' type.  ``residual_out`` and
    ``normalized`` may be given, also in the place of ``residual`` or ``delta``; rows of an output may not
    interleave with those of another tensor of the call.  Without ``delta`` the residual comes back as it is.
    """
    dtype = residual.dtype
    code = _DTYPES.get(dtype)
    if residual.dim() != 2 or code is None:
        raise ValueError("block_norm: residual must be [rows, width], bfloat16 or float32")
    if not residual.is_cuda:
        raise ValueError("block_norm: tensors must be on a CUDA device")
    shape, index = residual.shape, residual.get_device()
    rows, width = shape
    if delta is None and (post_weight is not None or gate is not None or residual_out is not None):
        raise ValueError("block_norm: post_weight, gate and residual_out need a delta")
    wdtype = norm_weight.dtype
    wcode = _DTYPES.get(wdtype)
    if wcode is None:
        raise ValueError("block_norm: norm_weight must be bfloat16 or float32")
    norm_w = _weight(norm_weight, width, index, "norm_weight")
    post_w = launch.NO_BUFFER
    if post_weight is not None:
        post_w = _weight(post_weight, width, index, "post_weight")
        if post_weight.dtype is not wdtype:
            raise ValueError("block_norm: norm_weight and post_weight must have one type")
    gate_buf, gate_rs, gate_cs = launch.NO_BUFFER, 0, 0
    if gate is not None:
        if gate.dim() != 2 or gate.shape[0] not in (1, rows) or gate.shape[1] not in (1, width):
            raise ValueError("block_norm: gate must be [rows, 1], [1, width] or [rows, width]")
        if gate.dtype is not dtype or gate.get_device() != index:
            raise ValueError("block_norm: gate must have the type and device of residual")
        gate_rs = gate.stride(0) if gate.shape[0] > 1 else 0
        gate_cs = gate.stride(1) if gate.shape[1] > 1 else 0
        if gate_cs > 1:
            raise ValueError("block_norm: gate must be contiguous along its rows")
        span = (gate.shape[0] - 1) * gate_rs + (gate.shape[1] - 1) * gate_cs + 1
        gate_buf = (gate.data_ptr(), span * _SIZES[dtype], 0, 0)
    res, res_stride = launch.rows_buffer(residual, rows, width, _SIZES[dtype], "block_norm: residual")
    whole = residual.is_contiguous()          # empty_like is the cheapest allocation
    if normalized is None:
        normalized = torch.empty_like(residual) if whole else residual.new_empty(shape)
        norm, norm_stride = (normalized.data_ptr(), rows * width * _SIZES[dtype], 0, 0), width
    else:
        norm, norm_stride = _rows(normalized, shape, dtype, index, "normalized")
    dlt, dlt_stride, out, out_stride = launch.NO_BUFFER, 0, launch.NO_BUFFER, 0
    if delta is not None:
        dlt, dlt_stride = _rows(delta, shape, dtype, index, "delta")
        if residual_out is None:
            residual_out = torch.empty_like(residual) if whole else residual.new_empty(shape)
            out, out_stride = (residual_out.data_ptr(), rows * width * _SIZES[dtype], 0, 0), width
        else:
            out, out_stride = _rows(residual_out, shape, dtype, index, "residual_out")
    if rows:
        launch.call(lib, "glmrt_b200_block_norm_async",
                    _ARGS.pack(*res, *dlt, *norm_w, *post_w, *gate_buf, *out, *norm,
                               rows, width, res_stride, dlt_stride, gate_rs, gate_cs, out_stride, norm_stride,
                               code, wcode, scale, eps), index)
    return (residual if delta is None else residual_out), normalized
