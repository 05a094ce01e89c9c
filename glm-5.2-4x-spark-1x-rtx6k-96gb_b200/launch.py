"""How the wrappers of the stateless operators reach the library.

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


def rows_buffer(t: torch.Tensor, rows: int, width: int) -> tuple[tuple, int]:
    """Packed fields and row stride (elements) of [rows, width] with rows contiguous inside."""
    stride = t.stride(0) if rows > 1 else width
    return (t.data_ptr(), ((rows - 1) * stride + width) * t.element_size() if rows else 0, 0, 0), stride


def call(lib: N.NativeLibrary | None, symbol: str, packed: bytes, device: torch.device) -> None:
    lib = lib or N.library()
    index = device.index
    if index == torch.cuda.current_device():
        lib.call(symbol, packed, C.c_void_p(torch._C._cuda_getCurrentRawStream(index)))
    else:
        with torch.cuda.device(index):
            lib.call(symbol, packed, C.c_void_p(torch._C._cuda_getCurrentRawStream(index)))


def check(lib: N.NativeLibrary | None = None) -> None:
    """Waits for the current stream and raises if a block norm or an 8-bit product on this device reported a wait
    that expired (glmrt_b200_operators_check)."""
    (lib or N.library()).call("glmrt_b200_operators_check", C.c_void_p(torch.cuda.current_stream().cuda_stream))
