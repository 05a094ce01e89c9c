"""How the wrappers of the operators around the routed experts reach the library.

A call's arguments travel as one packed struct (``struct.Struct`` costs a tenth of building ctypes objects
field by field), on the current stream of the tensors' device, with that device current.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import native as N

BUFFER = "PQi4xQ"              # glmrt_device_buffer_t: address, bytes, device, flags
NO_BUFFER = (0, 0, 0, 0)


def buffer(t: torch.Tensor | None) -> tuple:
    """Packed fields of a contiguous tensor (None: a null buffer)."""
    return NO_BUFFER if t is None else (t.data_ptr(), t.nbytes, 0, 0)


def rows_buffer(t: torch.Tensor, rows: int, width: int, size: int, what: str) -> tuple[tuple, int]:
    """Packed fields and row stride (elements) of [rows, width] with rows contiguous inside, `size` bytes a value."""
    if t.is_contiguous():
        return (t.data_ptr(), rows * width * size, 0, 0), width
    if width > 1 and t.stride(1) != 1:
        raise ValueError(f"{what} must be contiguous along its rows")
    if rows == 1:
        return (t.data_ptr(), width * size, 0, 0), width
    stride = t.stride(0)
    return (t.data_ptr(), ((rows - 1) * stride + width) * size, 0, 0), stride


def call(lib: N.NativeLibrary | None, symbol: str, packed: bytes, index: int, *handle) -> None:
    """``symbol(*handle, packed, current stream of device index)``; raises what NativeLibrary.call raises."""
    lib = lib or N.library()
    fn = lib.symbol(symbol)
    if index == torch._C._cuda_getDevice():
        stream = torch._C._cuda_getCurrentRawStream(index)
        status = fn(*handle, packed, C.c_void_p(stream) if stream else None)
    else:
        with torch.cuda.device(index):
            status = fn(*handle, packed, C.c_void_p(torch._C._cuda_getCurrentRawStream(index)))
    if status != 0:
        raise N.GlmrtError(symbol, status, lib.last_error())


def check(lib: N.NativeLibrary | None = None) -> None:
    """Waits for the current stream and raises if a block norm or an 8-bit product on this device reported a wait
    that expired (glmrt_b200_operators_check)."""
    (lib or N.library()).call("glmrt_b200_operators_check", C.c_void_p(torch.cuda.current_stream().cuda_stream))
