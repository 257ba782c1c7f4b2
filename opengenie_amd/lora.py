"""Low-rank adapters of many requests at once beside a shared projection, and
their backward pass, for the linears of `ltx_ops`. No counterpart in the
reference.

x (..., K) and y (..., N) are read as rows; rows segment_starts[s] ..
segment_starts[s + 1] - 1 belong to request s and take adapter
segment_adapters[s] (one outside 0 .. L - 1 is none; rows outside all segments
have none). Adapter l is a[l] [r, K], b[l] [N, r], scale[l]:

    y' = y + scale (x a^T) b^T
    dx = scale (dy b) a,  da = scale (dy b)^T x,  db = scale dy^T (x a^T)

with da and db summed over an adapter's rows, in a fixed order. The segments
stay on the device: nothing synchronises. Starts have to rise; the kernels
stay within the tensors whatever they hold.

On the GPU these run oga_lora_add and oga_lora_bwd on torch's current stream:
bf16 or fp16, r a multiple of 8 up to 128, K and N multiples of 8. Other
inputs take the same formulas in torch, in float32; under
OPENGENIE_AMD_STRICT=1 a GPU input that would do so raises. Tensors that do not
fit each other raise ValueError.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from ._launch import bytes_on, call_on, fresh, rows_layout, scratch
from .ltx_ops import _fallback, _hip, _xdt, fp8_linear_forward

_INDEX = (torch.int32, torch.int64)

__all__ = ["LoraAdapters", "lora_add", "lora_backward", "lora_add_with_grad", "fp8_linear_lora_forward"]


@dataclass
class LoraAdapters:
    """Adapters of one projection: a [L, r, K], b [L, N, r], scale [L] float32
    (None: 1)."""
    a: torch.Tensor
    b: torch.Tensor
    scale: torch.Tensor | None = None

    @staticmethod
    def stack(adapters: list[tuple[torch.Tensor, torch.Tensor, float]]) -> "LoraAdapters":
        """From (a [r, K], b [N, r], scale) of each adapter; smaller ranks are
        filled up with zeros to the largest one, to a multiple of 8."""
        rank = max((a.shape[0] + 7) // 8 * 8 for a, _, _ in adapters)
        pad = torch.nn.functional.pad
        return LoraAdapters(torch.stack([pad(a, (0, 0, 0, rank - a.shape[0])) for a, _, _ in adapters]),
                            torch.stack([pad(b, (0, rank - b.shape[1])) for _, b, _ in adapters]),
                            torch.tensor([float(s) for _, _, s in adapters], device=adapters[0][0].device))


def _check(x, n, a, b, scale, starts, ids):
    """(K, adapters, rank, segments) of a call whose tensors fit each other."""
    sa, sb, k, dtype, device = a.shape, b.shape, x.shape[-1], x.dtype, x.device
    if len(sa) != 3 or len(sb) != 3 or sa[0] != sb[0] or sa[1] != sb[2] or not sa[0] * sa[1] * sa[2]:
        raise ValueError(f"adapters a {tuple(sa)}, b {tuple(sb)}")
    if sa[2] != k or sb[1] != n:
        raise ValueError(f"adapters a {tuple(sa)}, b {tuple(sb)} for {k} -> {n}")
    if a.dtype != dtype or b.dtype != dtype or not dtype.is_floating_point:
        raise ValueError(f"dtypes x {dtype}, a {a.dtype}, b {b.dtype}")
    if scale is not None and (scale.shape != sa[:1] or scale.dtype != torch.float32):
        raise ValueError(f"scale {scale.dtype} {tuple(scale.shape)} of {sa[0]} adapters")
    ss, si = starts.shape, ids.shape
    if (len(ss) != 1 or len(si) != 1 or ss[0] != si[0] + 1 or starts.dtype not in _INDEX or ids.dtype not in _INDEX):
        raise ValueError(f"segments: starts {starts.dtype} {tuple(ss)}, adapters {ids.dtype} {tuple(si)}")
    if (a.device != device or b.device != device or starts.device != device or ids.device != device
            or (scale is not None and scale.device != device)):
        raise ValueError("adapter inputs on different devices")
    return k, sa[0], sa[1], si[0]


def _kernel_ok(x, n, k, rank, adapters) -> bool:
    return (x.is_cuda and (x.dtype == torch.bfloat16 or x.dtype == torch.float16) and rank % 8 == 0 and rank <= 128
            and k % 8 == 0 and n % 8 == 0 and adapters <= 2000)


def _i32(t: torch.Tensor, most: int) -> torch.Tensor:
    if t.dtype != torch.int32:
        t = t.clamp(-1, most).to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def _packed(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() and not t.data_ptr() & 15 else t.clone(memory_format=torch.contiguous_format)


def _torch_rows(x, a, starts, ids, scale):
    """For each row and adapter whether the row takes it [T, L], and the scale
    of each of the L r ranks."""
    row = torch.arange(x.shape[0], device=x.device)
    seg = torch.searchsorted(starts.long().contiguous(), row, right=True) - 1
    inside = (seg >= 0) & (seg < ids.shape[0])
    mine = torch.where(inside, ids.long()[seg.clamp(0, max(ids.shape[0] - 1, 0))], -1) if ids.shape[0] else row * 0 - 1
    keep = mine[:, None] == torch.arange(a.shape[0], device=x.device)
    s = torch.ones(a.shape[0], device=x.device) if scale is None else scale
    return keep.repeat_interleave(a.shape[1], 1), s.repeat_interleave(a.shape[1])


def _torch_low(x, w, keep, s):
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    return torch.where(keep, torch.matmul(x.to(wide), w.to(wide)) * s.to(wide), 0.0)


def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor | None,
             segment_starts: torch.Tensor, segment_adapters: torch.Tensor, *, out: torch.Tensor | None = None,
             save_low: bool = False):
    """y + scale (x a^T) b^T row by row, into `out` (which may be y) or a new
    tensor; with `save_low` also the rows' scale (x a^T), which
    `lora_backward` reads."""
    shape = y.shape
    n = shape[-1]
    k, adapters, rank, segments = _check(x, n, a, b, scale, segment_starts, segment_adapters)
    if shape[:-1] != x.shape[:-1] or y.dtype != x.dtype or y.device != x.device:
        raise ValueError(f"y {y.dtype} {tuple(shape)} for x {x.dtype} {tuple(x.shape)}")
    if out is not None and (out.shape != y.shape or out.dtype != y.dtype or out.device != y.device
                            or not out.is_contiguous()):
        raise ValueError(f"out {out.dtype} {tuple(out.shape)} for y {y.dtype} {tuple(y.shape)}, contiguous")
    rows = x.numel() // k
    if rows == 0 or segments == 0:
        r = y.clone(memory_format=torch.contiguous_format) if out is None else out if out is y else out.copy_(y)
        return (r, torch.zeros((rows, rank), device=x.device, dtype=torch.float32)) if save_low else r
    if not _kernel_ok(x, n, k, rank, adapters) or (out is not None and out.data_ptr() % 16):
        _fallback("lora_add", y, x)
        x2 = x.reshape(-1, k)
        keep, s = _torch_rows(x2, a, segment_starts, segment_adapters, scale)
        low = _torch_low(x2, a.flatten(0, 1).t(), keep, s)
        r = y.reshape(-1, n).to(low.dtype) + torch.matmul(low, b.to(low.dtype).transpose(1, 2).flatten(0, 1))
        r = r.to(y.dtype).reshape(y.shape)
        r = r if out is None else out.copy_(r)
        return (r, low.reshape(rows, -1, rank).sum(1)) if save_low else r
    if out is None:
        out = fresh(y)
    x2, xs = rows_layout(x)
    y2, ys = rows_layout(y)
    low = x.new_empty((rows, rank), dtype=torch.float32) if save_low else None
    a, b = _packed(a), _packed(b)
    scale = scale if scale is None or scale.is_contiguous() else scale.contiguous()
    starts, ids = _i32(segment_starts, rows), _i32(segment_adapters, adapters)
    size = bytes_on(x, "oga_lora_add_workspace_bytes", rows, k, rank, segments)
    ws = scratch(x, size)
    _hip("lora_add")
    call_on(x, "oga_lora_add", _xdt(x), y2.data_ptr(), ys, x2.data_ptr(), xs, a.data_ptr(), b.data_ptr(),
            None if scale is None else scale.data_ptr(), starts.data_ptr(), ids.data_ptr(), segments, adapters,
            None if low is None else low.data_ptr(), out.data_ptr(), n, rows, k, n, rank, ws.data_ptr(), size)
    return (out, low) if save_low else out


def lora_backward(dy: torch.Tensor, x: torch.Tensor, low: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                  scale: torch.Tensor | None, segment_starts: torch.Tensor, segment_adapters: torch.Tensor):
    """dx, da, db of `lora_add` with these inputs from its output's gradient
    and the `low` it saved (y's gradient is dy)."""
    n = dy.shape[-1]
    k, adapters, rank, segments = _check(x, n, a, b, scale, segment_starts, segment_adapters)
    if dy.shape[:-1] != x.shape[:-1] or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError(f"dy {dy.dtype} {tuple(dy.shape)} for x {x.dtype} {tuple(x.shape)}")
    rows = x.numel() // k
    if low.shape != (rows, rank) or low.device != x.device or not low.is_floating_point():
        raise ValueError(f"low {low.dtype} {tuple(low.shape)} of {rows} rows, rank {rank}")
    if rows == 0 or segments == 0:
        return torch.zeros(x.shape, device=x.device, dtype=x.dtype), torch.zeros_like(a), torch.zeros_like(b)
    if not _kernel_ok(x, n, k, rank, adapters) or low.dtype != torch.float32:
        _fallback("lora_backward", dy, x)
        x2, dy2 = x.reshape(-1, k), dy.reshape(-1, n)
        keep, s = _torch_rows(x2, a, segment_starts, segment_adapters, scale)
        dlow = _torch_low(dy2, b.transpose(1, 2).flatten(0, 1).t(), keep, s)
        mine = torch.where(keep, low.to(dlow.dtype).repeat(1, a.shape[0]), 0.0)
        some = keep.any(1, keepdim=True)
        xf, df = (torch.where(some, t.to(dlow.dtype), 0.0) for t in (x2, dy2))
        dx = torch.matmul(dlow, a.to(dlow.dtype).flatten(0, 1)).to(x.dtype).reshape(x.shape)
        da = torch.matmul(dlow.t(), xf).reshape(a.shape).to(a.dtype)
        db = torch.matmul(mine.t(), df).reshape(a.shape[0], rank, n).transpose(1, 2).contiguous().to(b.dtype)
        return dx, da, db
    dx = fresh(x)
    x2, xs = rows_layout(x)
    dy2, dys = rows_layout(dy)
    low, a, b = _packed(low), _packed(a), _packed(b)
    scale = scale if scale is None or scale.is_contiguous() else scale.contiguous()
    starts, ids = _i32(segment_starts, rows), _i32(segment_adapters, adapters)
    da, db = torch.empty_like(a), torch.empty_like(b)
    size = bytes_on(x, "oga_lora_bwd_workspace_bytes", rows, k, n, rank, adapters, segments)
    ws = scratch(x, size)
    _hip("lora_backward")
    call_on(x, "oga_lora_bwd", _xdt(x), dy2.data_ptr(), dys, x2.data_ptr(), xs, low.data_ptr(), a.data_ptr(),
            b.data_ptr(), None if scale is None else scale.data_ptr(), starts.data_ptr(), ids.data_ptr(),
            segments, adapters, dx.data_ptr(), k, da.data_ptr(), db.data_ptr(), rows, k, n, rank, ws.data_ptr(),
            size)
    return dx, da, db


class _LoraAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, a, b, scale, segment_starts, segment_adapters):
        r, low = lora_add(y, x, a, b, scale, segment_starts, segment_adapters, save_low=True)
        ctx.save_for_backward(x, low, a, b, scale, segment_starts, segment_adapters)
        return r

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, low, a, b, scale, starts, ids = ctx.saved_tensors
        return (dy, *lora_backward(dy, x, low, a, b, scale, starts, ids), None, None, None)


def lora_add_with_grad(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                       scale: torch.Tensor | None, segment_starts: torch.Tensor,
                       segment_adapters: torch.Tensor) -> torch.Tensor:
    """`lora_add`, differentiable in y, x, a and b."""
    return _LoraAdd.apply(y, x, a, b, scale, segment_starts, segment_adapters)


def fp8_linear_lora_forward(module, x: torch.Tensor, adapters: LoraAdapters, segment_starts: torch.Tensor,
                            segment_adapters: torch.Tensor) -> torch.Tensor:
    """`ltx_ops.fp8_linear_forward(module, x)` with the requests' adapters
    added to its output in place."""
    y = fp8_linear_forward(module, x)
    return lora_add(y, x, adapters.a, adapters.b, adapters.scale, segment_starts, segment_adapters,
                    out=y if y.is_contiguous() else None)
