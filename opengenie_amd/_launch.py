"""What the operators with a row layout of their own share: layouts the kernels
read, and a call on the tensors' own device and current stream."""

from __future__ import annotations

import torch

from . import _lib
from .ltx_ops import _stream


_device = torch._C._cuda_getDevice


def call_on(t: torch.Tensor, name: str, *args) -> None:
    """_lib.call(name, *args, stream) on t's device and its current stream."""
    index = t.get_device()
    if _device() == index:
        _lib.call(name, *args, _stream(t))
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args, _stream(t))


def bytes_on(t: torch.Tensor, name: str, *args) -> int:
    """A workspace query, which may go by t's device."""
    index = t.get_device()
    if _device() == index:
        return _lib.function(name)(*args)
    with torch.cuda.device(index):
        return _lib.function(name)(*args)


def fresh(t: torch.Tensor) -> torch.Tensor:
    """An empty contiguous tensor of t's shape, dtype and device (empty_like
    takes half of empty's time with all of them named)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def scratch(t: torch.Tensor, size: int) -> torch.Tensor:
    """size bytes, an even number, on the device of t, a 16-bit tensor (in its
    own dtype, which new_empty need not be told)."""
    return t.new_empty(size >> 1)


def heads_layout(t: torch.Tensor, most: int = 1 << 62) -> tuple[torch.Tensor, tuple[int, int, int]]:
    """t [B, N, H, D] as the kernels read it, and its (batch, token, head)
    strides: unit stride along D, 16-byte aligned rows, token and head strides
    below `most`; a copy where t is laid out otherwise (an expanded gradient, a
    transposed view, an odd offset). An axis of one element has stride 0."""
    sb, sn, sh, sd = t.stride()
    if sd == 1 and not (sb | sn | sh) & 7 and 0 <= sn < most and 0 <= sh < most and not t.data_ptr() & 15:
        return t, (sb, sn, sh)
    b, n, h, d = t.shape
    sb, sn, sh = sb if b > 1 else 0, sn if n > 1 else 0, sh if h > 1 else 0
    if (sd != 1 and d > 1) or (sb | sn | sh) & 7 or t.data_ptr() & 15 or not 0 <= sn < most or not 0 <= sh < most:
        t = t.clone(memory_format=torch.contiguous_format)
        sb, sn, sh = n * h * d, h * d, d
    return t, (sb, sn, sh)


def rows_layout(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """t (..., C) as rows of C, and the row stride: unit stride along C,
    16-byte aligned rows, strides below 2^25; a copy where t is laid out
    otherwise."""
    if t.ndim != 2:
        t = t.reshape(-1, t.shape[-1])
    stride, unit = t.stride()
    if unit != 1 or stride & 7 or stride >= 1 << 25 or t.data_ptr() & 15:
        if t.shape[0] == 1 and (unit == 1 or t.shape[1] == 1) and not t.data_ptr() & 15:
            return t, 0
        t = t.clone(memory_format=torch.contiguous_format)
        stride = t.stride(0)
    return t, stride


def vector32(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """t as a contiguous vector of dtype on a 32-byte boundary."""
    if t.dtype != dtype:
        t = t.to(dtype)
    if not t.is_contiguous() or t.data_ptr() & 31:
        t = t.clone(memory_format=torch.contiguous_format)
    return t
