"""Residual add and RMSNorms at the boundary of a block, in one kernel (csrc/norm.cu).

The routed layer takes rows that are already normalised; this makes them, together with the new
residual stream (python/reference/glmrt_reference/glm_moe_dsa_layer_ref.py:157-206):

    d = delta;  d *= rsqrt(mean(d^2) + eps) * post_weight;  d *= gate        (each where given)
    r = residual + scale * d
    y = r * rsqrt(mean(r^2) + eps) * norm_weight
"""
from __future__ import annotations

import ctypes as C

import torch

from . import native as N

_DTYPES = {torch.bfloat16: N.DTYPE_BF16, torch.float32: N.DTYPE_F32}


def _rows(t: torch.Tensor, like: torch.Tensor, what: str) -> tuple[N.DeviceBuffer, int]:
    """Buffer and row stride of a [rows, width] tensor whose rows are contiguous inside."""
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"block_norm: {what} must have the shape, type and device of residual")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"block_norm: {what} must be contiguous along its rows")
    rows, width = t.shape
    stride = t.stride(0) if rows > 1 else width
    nbytes = ((rows - 1) * stride + width) * t.element_size() if rows else 0
    return N.DeviceBuffer.of(t.data_ptr(), nbytes, t.device.index), stride


def block_norm(residual: torch.Tensor, delta: torch.Tensor | None = None, *, norm_weight: torch.Tensor,
               post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
               eps: float = 1e-5, residual_out: torch.Tensor | None = None, normalized: torch.Tensor | None = None,
               lib: N.NativeLibrary | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(residual + scale * branch, its RMSNorm)``; rows bf16 or float32, weights bf16 or float32.

    ``gate``: [rows, 1], [1, width] or [rows, width] of the rows' type.  ``residual_out`` and
    ``normalized`` may be given, also in the place of ``residual`` or ``delta``.  Without ``delta``
    the residual comes back as it is.
    """
    if residual.dim() != 2 or residual.dtype not in _DTYPES:
        raise ValueError("block_norm: residual must be [rows, width], bfloat16 or float32")
    if not residual.is_cuda:
        raise ValueError("block_norm: tensors must be on a CUDA device")
    rows, width = residual.shape
    if delta is None and (post_weight is not None or gate is not None or residual_out is not None):
        raise ValueError("block_norm: post_weight, gate and residual_out need a delta")
    a = N.BlockNormArgs()
    a.rows, a.width, a.scale, a.eps = rows, width, scale, eps
    a.dtype = _DTYPES[residual.dtype]
    for name, w in (("norm_weight", norm_weight), ("post_weight", post_weight)):
        if w is None:
            continue
        if w.shape != (width,) or w.dtype not in _DTYPES or w.device != residual.device or not w.is_contiguous():
            raise ValueError(f"block_norm: {name} must be a contiguous [{width}] bfloat16 or float32 tensor on the rows' device")
        if w.dtype != norm_weight.dtype:
            raise ValueError("block_norm: norm_weight and post_weight must have one type")
        setattr(a, name, N.DeviceBuffer.of(w.data_ptr(), width * w.element_size(), w.device.index))
    a.weight_dtype = _DTYPES[norm_weight.dtype]
    if gate is not None:
        if gate.dim() != 2 or gate.shape[0] not in (1, rows) or gate.shape[1] not in (1, width):
            raise ValueError("block_norm: gate must be [rows, 1], [1, width] or [rows, width]")
        if gate.dtype != residual.dtype or gate.device != residual.device:
            raise ValueError("block_norm: gate must have the type and device of residual")
        a.gate_row_stride = gate.stride(0) if gate.shape[0] > 1 else 0
        a.gate_col_stride = gate.stride(1) if gate.shape[1] > 1 else 0
        if a.gate_col_stride > 1:
            raise ValueError("block_norm: gate must be contiguous along its rows")
        span = (gate.shape[0] - 1) * a.gate_row_stride + (gate.shape[1] - 1) * a.gate_col_stride + 1
        if a.gate_col_stride == 0 and gate.shape[1] == width and width > 1:
            span = (gate.shape[0] - 1) * a.gate_row_stride + 1          # an expanded column
        a.gate = N.DeviceBuffer.of(gate.data_ptr(), span * gate.element_size(), gate.device.index)
    if normalized is None:
        normalized = torch.empty((rows, width), dtype=residual.dtype, device=residual.device)
    a.residual, a.residual_stride = _rows(residual, residual, "residual")
    a.normalized, a.normalized_stride = _rows(normalized, residual, "normalized")
    if delta is not None:
        if residual_out is None:
            residual_out = torch.empty((rows, width), dtype=residual.dtype, device=residual.device)
        a.delta, a.delta_stride = _rows(delta, residual, "delta")
        a.residual_out, a.residual_out_stride = _rows(residual_out, residual, "residual_out")
    if rows:
        with torch.cuda.device(residual.device):
            (lib or N.library()).call("glmrt_b200_block_norm_async", C.byref(a),
                                      C.c_void_p(torch.cuda.current_stream().cuda_stream))
    return (residual if delta is None else residual_out), normalized
