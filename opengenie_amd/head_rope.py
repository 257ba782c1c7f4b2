"""RMSNorm of each query and key head with the position rotation, its backward
pass, and the rotation alone, beside the whole-row norms of
`ltx_ops.fused_video_qk_rmsnorm_rope`. No counterpart in the reference.

q [B, N, H, D], k [B, N, Hk, D]; per head y = Rot(x r w), r =
1/sqrt(mean(x^2) + eps), w [D] (None: no weight). Rot turns the first R = 2 *
cos.shape[-1] elements of each head by the token's angles, in planes (i, i +
R/2) with layout "half" or (2i, 2i + 1) with "interleaved"; the others pass.
cos and sin [P, R/2] (`rope.rotary_cos_sin`) have a row per position: token n's
is row n, or row positions[b, n] (a position outside the tables reads their
first or last row). Everything is float32, rounded once.

On the GPU these run oga_head_rmsnorm_rope and oga_head_rmsnorm_rope_bwd on
torch's current stream: bf16 or fp16 heads of 64, 128 or 256, R a multiple of
16, bf16 or float32 weights and tables. Other inputs take the same formulas in
torch; under OPENGENIE_AMD_STRICT=1 a GPU input that would do so raises.
Tensors that do not fit each other raise ValueError.
"""

from __future__ import annotations

import torch

from ._launch import bytes_on, call_on, fresh, heads_layout, scratch, vector32
from .ltx_ops import _any_dt, _fallback, _hip, _xdt

__all__ = ["qk_head_rmsnorm_rope", "qk_head_rmsnorm_rope_backward", "qk_head_rmsnorm_rope_with_grad", "apply_rope"]

_PARAM = (torch.bfloat16, torch.float32)


def _check(x, k, cos, sin, layout, positions) -> None:
    if layout != "half" and layout != "interleaved":
        raise ValueError(f"unknown rotary layout: {layout}")
    shape, dtype, device, table = x.shape, x.dtype, x.device, cos.shape
    if len(shape) != 4 or not dtype.is_floating_point:
        raise ValueError(f"heads {dtype} {tuple(shape)}")
    if k is not None:
        other = k.shape
        if (len(other) != 4 or other[0] != shape[0] or other[1] != shape[1] or other[3] != shape[3]
                or k.dtype != dtype or k.device != device):
            raise ValueError(f"k {k.dtype} {tuple(other)} beside q {dtype} {tuple(shape)}")
    if len(table) != 2 or table != sin.shape or cos.dtype != sin.dtype or not 0 < 2 * table[1] <= shape[3]:
        raise ValueError(f"cos {tuple(table)}, sin {tuple(sin.shape)} for heads of {shape[3]}")
    if cos.device != device or sin.device != device:
        raise ValueError("cos/sin on another device")
    if positions is None:
        if table[0] < shape[1]:
            raise ValueError(f"cos/sin of {table[0]} positions for {shape[1]} tokens")
    else:
        if positions.shape != shape[:2] or (positions.dtype != torch.int32 and positions.dtype != torch.int64):
            raise ValueError(f"positions {positions.dtype} {tuple(positions.shape)} for {tuple(shape[:2])} tokens")
        if positions.device != device:
            raise ValueError("positions on another device")
        if table[0] < 1:
            raise ValueError("cos/sin without positions")


def _check_weight(q, w) -> None:
    if w is not None and (w.shape != q.shape[3:] or w.device != q.device or not w.dtype.is_floating_point):
        raise ValueError(f"weight {w.dtype} {tuple(w.shape)} for heads of {q.shape[3]}")


def _kernel_ok(x, cos, q_weight=None, k_weight=None) -> bool:
    return (x.is_cuda and (x.dtype == torch.bfloat16 or x.dtype == torch.float16) and x.shape[3] in (64, 128, 256)
            and cos.shape[1] % 8 == 0 and cos.dtype in _PARAM and (q_weight is None or q_weight.dtype in _PARAM)
            and (k_weight is None or k_weight.dtype in _PARAM))


def _tables(cos, sin):
    """Tables with rows the kernel reads 4 entries at a time, and their row
    stride."""
    (row, unit), other = cos.stride(), sin.stride()
    if unit != 1 or row & 3 or row < 0 or other != (row, 1) or cos.data_ptr() & 15 or sin.data_ptr() & 15:
        cos, sin = (t.clone(memory_format=torch.contiguous_format) for t in (cos, sin))
        row = cos.shape[1]
    return cos, sin, row


def _weights(q_weight, k_weight):
    """Both weights as the kernels read them in one dtype: theirs, or float32
    where they differ."""
    if q_weight is None and k_weight is None:
        return None, None, torch.float32
    dtype = (k_weight if q_weight is None else q_weight).dtype
    if q_weight is not None and k_weight is not None and k_weight.dtype != dtype:
        dtype = torch.float32
    return (None if q_weight is None else vector32(q_weight, dtype),
            None if k_weight is None else vector32(k_weight, dtype), dtype)


def _pos_args(positions):
    if positions is None:
        return None, 0, (0, 0)
    return positions.data_ptr(), int(positions.dtype == torch.int64), positions.stride()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _torch_tables(cos, sin, n, positions, dt):
    if positions is None:
        return cos[:n].to(dt)[None, :, None, :], sin[:n].to(dt)[None, :, None, :]
    at = positions.long().clamp(0, cos.shape[0] - 1)
    return cos[at].to(dt)[:, :, None, :], sin[at].to(dt)[:, :, None, :]


def _torch_turn(x, cos, sin, layout):
    half = cos.shape[-1]
    if layout == "half":
        a, b = x[..., :half], x[..., half:2 * half]
        head = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        head = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((head, x[..., 2 * half:]), -1)


def _wide(x):
    return torch.float64 if x.dtype == torch.float64 else torch.float32


def _torch_norm_turn(x, w, eps, cos, sin, layout):
    xf = x.to(_wide(x))
    n = xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + eps)
    return _torch_turn(n if w is None else n * w.to(xf.dtype), cos, sin, layout).to(x.dtype)


def _torch_norm_turn_grad(dy, x, w, eps, cos, sin, layout):
    xf = x.to(_wide(x))
    r = torch.rsqrt(xf.square().mean(-1, keepdim=True) + eps)
    dn = _torch_turn(dy.to(xf.dtype), cos, -sin, layout)
    n = xf * r
    dw = None if w is None else (dn * n).sum((0, 1, 2)).to(w.dtype)
    g = dn if w is None else dn * w.to(xf.dtype)
    return (r * (g - n * (g * n).mean(-1, keepdim=True))).to(x.dtype), dw


def _forward(q, k, q_weight, k_weight, eps, cos, sin, layout, positions, norm, inverse):
    b, n, h, d = q.shape
    q, qs = heads_layout(q)
    q_out = fresh(q)
    hk, k_out, kp, kop, ks, kos = 0, None, None, None, (0, 0, 0), (0, 0, 0)
    if k is not None:
        hk = k.shape[2]
        k, ks = heads_layout(k)
        k_out = fresh(k)
        kos = (n * hk * d, hk * d, d)
        kp, kop = k.data_ptr(), k_out.data_ptr()
    qw, kw, wdt = _weights(q_weight, k_weight)
    cos, sin, row = _tables(cos, sin)
    pos, pos64, pos_strides = _pos_args(positions)
    length, half = cos.shape
    call_on(q, "oga_head_rmsnorm_rope", _xdt(q), q.data_ptr(), qs, kp, ks, _ptr(qw), _ptr(kw),
            0 if wdt == torch.bfloat16 else 1, cos.data_ptr(), sin.data_ptr(), _any_dt(cos), row, length, pos, pos64,
            pos_strides, q_out.data_ptr(), (n * h * d, h * d, d), kop, kos, b, n, h, hk, d, 2 * half,
            layout == "interleaved", inverse, norm, eps)
    return q_out, k_out


def qk_head_rmsnorm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None,
                         k_weight: torch.Tensor | None, eps: float, cos: torch.Tensor, sin: torch.Tensor, *,
                         layout: str = "half", positions: torch.Tensor | None = None):
    """The normed and rotated q and k, in one pass over both."""
    _check(q, k, cos, sin, layout, positions)
    _check_weight(q, q_weight)
    _check_weight(q, k_weight)
    if not (q.numel() and k.numel() and _kernel_ok(q, cos, q_weight, k_weight)):
        if q.numel() and k.numel():
            _fallback("qk_head_rmsnorm_rope", q, k)
        c, s = _torch_tables(cos, sin, q.shape[1], positions, _wide(q))
        return (_torch_norm_turn(q, q_weight, eps, c, s, layout), _torch_norm_turn(k, k_weight, eps, c, s, layout))
    _hip("qk_head_rmsnorm_rope")
    return _forward(q, k, q_weight, k_weight, float(eps), cos, sin, layout, positions, True, False)


def qk_head_rmsnorm_rope_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                                  q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, eps: float,
                                  cos: torch.Tensor, sin: torch.Tensor, *, layout: str = "half",
                                  positions: torch.Tensor | None = None):
    """dq, dk, dq_weight, dk_weight (None where there is no weight) of
    `qk_head_rmsnorm_rope` with these inputs, from its outputs' gradients. The
    weights' gradients are summed without atomics, in a fixed order."""
    _check(q, k, cos, sin, layout, positions)
    _check_weight(q, q_weight)
    _check_weight(q, k_weight)
    for g, x in ((dq_out, q), (dk_out, k)):
        if g.shape != x.shape or g.dtype != x.dtype or g.device != x.device:
            raise ValueError(f"gradient {g.dtype} {tuple(g.shape)} of {x.dtype} {tuple(x.shape)}")
    if not (q.numel() and k.numel() and _kernel_ok(q, cos, q_weight, k_weight)):
        if q.numel() and k.numel():
            _fallback("qk_head_rmsnorm_rope_backward", q, k)
        c, s = _torch_tables(cos, sin, q.shape[1], positions, _wide(q))
        dq, dqw = _torch_norm_turn_grad(dq_out, q, q_weight, eps, c, s, layout)
        dk, dkw = _torch_norm_turn_grad(dk_out, k, k_weight, eps, c, s, layout)
        return dq, dk, dqw, dkw
    _hip("qk_head_rmsnorm_rope_backward")
    b, n, h, d = q.shape
    hk = k.shape[2]
    q, qs = heads_layout(q)
    k, ks = heads_layout(k)
    dq_out, dqos = heads_layout(dq_out)
    dk_out, dkos = heads_layout(dk_out)
    dq, dk = fresh(q), fresh(k)
    qw, kw, wdt = _weights(q_weight, k_weight)
    dqw, dkw = (None if w is None else torch.empty((d,), device=q.device, dtype=wdt) for w in (qw, kw))
    cos, sin, row = _tables(cos, sin)
    pos, pos64, pos_strides = _pos_args(positions)
    ws, size = None, 0
    if qw is not None or kw is not None:
        size = bytes_on(q, "oga_head_rmsnorm_rope_bwd_workspace_bytes", d)
        ws = scratch(q, size)
    call_on(q, "oga_head_rmsnorm_rope_bwd", _xdt(q), dq_out.data_ptr(), dqos, dk_out.data_ptr(), dkos, q.data_ptr(),
            qs, k.data_ptr(), ks, _ptr(qw), _ptr(kw), 0 if wdt == torch.bfloat16 else 1, cos.data_ptr(),
            sin.data_ptr(), _any_dt(cos), row, cos.shape[0], pos, pos64, pos_strides, dq.data_ptr(),
            (n * h * d, h * d, d), dk.data_ptr(), (n * hk * d, hk * d, d), _ptr(dqw), _ptr(dkw), b, n, h, hk, d,
            2 * cos.shape[1], int(layout == "interleaved"), float(eps), _ptr(ws), size)
    if dqw is not None and dqw.dtype != q_weight.dtype:
        dqw = dqw.to(q_weight.dtype)
    if dkw is not None and dkw.dtype != k_weight.dtype:
        dkw = dkw.to(k_weight.dtype)
    return dq, dk, dqw, dkw


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *, layout: str = "half",
               positions: torch.Tensor | None = None, inverse: bool = False) -> torch.Tensor:
    """The rotation alone, x [B, N, H, D]; `inverse` turns back, which is also
    its backward pass."""
    _check(x, None, cos, sin, layout, positions)
    if x.numel() == 0 or not _kernel_ok(x, cos):
        if x.numel():
            _fallback("apply_rope", x)
        c, s = _torch_tables(cos, sin, x.shape[1], positions, _wide(x))
        return _torch_turn(x.to(_wide(x)), c, -s if inverse else s, layout).to(x.dtype)
    _hip("apply_rope")
    return _forward(x, None, None, None, 0.0, cos, sin, layout, positions, False, inverse)[0]


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, eps, cos, sin, layout, positions):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.how = eps, layout
        return qk_head_rmsnorm_rope(q, k, q_weight, k_weight, eps, cos, sin, layout=layout, positions=positions)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        eps, layout = ctx.how
        grads = qk_head_rmsnorm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, eps, cos, sin, layout=layout,
                                              positions=positions)
        return (*grads, None, None, None, None, None)


def qk_head_rmsnorm_rope_with_grad(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None,
                                   k_weight: torch.Tensor | None, eps: float, cos: torch.Tensor, sin: torch.Tensor,
                                   *, layout: str = "half", positions: torch.Tensor | None = None):
    """`qk_head_rmsnorm_rope`, differentiable in q, k and the weights."""
    return _NormRope.apply(q, k, q_weight, k_weight, eps, cos, sin, layout, positions)
