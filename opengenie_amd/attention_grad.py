"""Attention that is trained, beside the inference attention of
`opengenie_amd.attention`: the forward pass with each row's log-sum-exp, the
backward pass that recomputes the probabilities from it, and the two as one
differentiable call. No counterpart in the reference, which only infers.

q, out, dout [B, Nq, H, D], k, v [B, Nk, Hk, D], bf16, D 64 or 128; H a
multiple of Hk, each key head serving H / Hk query heads. `k_lens` [B] gives
the valid keys of each sequence of a padded batch (prompts of different
lengths); what k and v hold behind them is not read. With `causal` query i
sees the keys j <= i + k_lens[b] - Nq. A query that sees no key gives 0, has
lse -inf and no gradient; keys that no query sees have gradient 0.

On the GPU these run oga_attention_lse and oga_attention_bwd on torch's
current stream. Inputs the kernels do not cover (CPU tensors, other dtypes and
head dimensions) take the same formulas in torch, in float32 (float64 inputs in
float64); under OPENGENIE_AMD_STRICT=1 a GPU input that would do so raises.
Tensors that do not fit each other raise ValueError.
"""

from __future__ import annotations

import math

import torch

from ._launch import bytes_on, call_on, fresh, heads_layout, scratch
from .ltx_ops import _fallback, _hip

__all__ = ["flash_attn_lse", "flash_attn_backward", "attention_with_grad"]

_MOST = 1 << 24  # token strides the kernels take


def _check(q, k, v, k_lens):
    """The shapes (b, nq, h, d, nk, hk) of a call whose tensors fit each other."""
    qs, ks, dtype, device = q.shape, k.shape, q.dtype, q.device
    if len(qs) != 4 or len(ks) != 4 or ks != v.shape:
        raise ValueError(f"attention shapes q {tuple(qs)}, k {tuple(ks)}, v {tuple(v.shape)}")
    b, nq, h, d = qs
    kb, nk, hk, kd = ks
    if b != kb or d != kd or not hk or h % hk:
        raise ValueError(f"attention shapes q {tuple(qs)}, k {tuple(ks)}")
    if dtype != k.dtype or dtype != v.dtype or not dtype.is_floating_point:
        raise ValueError(f"attention dtypes q {dtype}, k {k.dtype}, v {v.dtype}")
    if device != k.device or device != v.device:
        raise ValueError("attention inputs on different devices")
    if k_lens is not None:
        if k_lens.shape != (b,) or (k_lens.dtype != torch.int32 and k_lens.dtype != torch.int64):
            raise ValueError(f"k_lens {k_lens.dtype} {tuple(k_lens.shape)} for a batch of {b}")
        if k_lens.device != device:
            raise ValueError("k_lens on another device")
    return b, nq, h, d, nk, hk


def _check_grad(dout, q, out, lse) -> None:
    shape, dtype, device = q.shape, q.dtype, q.device
    if dout.shape != shape or out.shape != shape or dout.dtype != dtype or out.dtype != dtype:
        raise ValueError(f"dout {dout.dtype} {tuple(dout.shape)}, out {out.dtype} {tuple(out.shape)} for q {dtype} "
                         f"{tuple(shape)}")
    if lse.shape != (shape[0], shape[2], shape[1]):
        raise ValueError(f"lse {tuple(lse.shape)} for q {tuple(shape)}")
    if dout.device != device or out.device != device or lse.device != device:
        raise ValueError("attention inputs on different devices")


def _kernel_ok(q, d: int, scale: float) -> bool:
    return q.is_cuda and q.dtype == torch.bfloat16 and (d == 64 or d == 128) and 0.0 < scale < 1e30


def _lens32(k_lens: torch.Tensor | None, nk: int) -> torch.Tensor | None:
    if k_lens is None:
        return None
    if k_lens.dtype != torch.int32:
        k_lens = k_lens.clamp(0, nk).to(torch.int32)
    return k_lens if k_lens.is_contiguous() else k_lens.contiguous()


def _torch_inputs(q, k, v, causal, k_lens):
    """q, k, v as [B, H, N, D] in float32 (or float64), keys behind their
    sequence zeroed, and the mask of hidden scores (None: none)."""
    dt = torch.float64 if q.dtype == torch.float64 else torch.float32
    group, nq, nk = q.shape[2] // k.shape[2], q.shape[1], k.shape[1]
    qf, kf, vf = (t.to(dt).transpose(1, 2) for t in (q, k, v))
    hide = None
    if k_lens is not None or causal:
        j = torch.arange(nk, device=q.device)
        lens = (k_lens.long().clamp(0, nk) if k_lens is not None
                else torch.full((q.shape[0],), nk, device=q.device)).view(-1, 1, 1, 1)
        hide = j >= lens
        kf, vf = (t.masked_fill(hide.transpose(2, 3), 0.0) for t in (kf, vf))
        if causal:
            hide = hide | (j > torch.arange(nq, device=q.device)[:, None] + lens - nq)
    kf, vf = (t.repeat_interleave(group, 1) for t in (kf, vf))
    return qf, kf, vf, hide


def _torch_lse(q, k, v, scale, causal, k_lens):
    qf, kf, vf, hide = _torch_inputs(q, k, v, causal, k_lens)
    s = torch.matmul(qf, kf.transpose(2, 3).contiguous()) * scale
    if hide is not None:
        s = s.masked_fill(hide, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
    return torch.matmul(p, vf).transpose(1, 2).contiguous().to(q.dtype), lse


def _torch_backward(dout, q, k, v, lse, scale, causal, k_lens):
    qf, kf, vf, hide = _torch_inputs(q, k, v, causal, k_lens)
    do = dout.to(qf.dtype).transpose(1, 2)
    s = torch.matmul(qf, kf.transpose(2, 3).contiguous()) * scale
    if hide is not None:
        s = s.masked_fill(hide, -math.inf)
    lse = lse.to(qf.dtype)
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dp = torch.matmul(do, vf.transpose(2, 3).contiguous())
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale  # (without out, which is rounded)
    dq, dk = torch.matmul(ds, kf), torch.matmul(ds.transpose(2, 3).contiguous(), qf)
    hk = k.shape[2]
    dk, dv = (t.unflatten(1, (hk, q.shape[2] // hk)).sum(2) for t in (dk, dv))
    return tuple(t.transpose(1, 2).contiguous().to(q.dtype) for t in (dq, dk, dv))


def flash_attn_lse(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, softmax_scale: float | None = None,
                   causal: bool = False, k_lens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """out [B, Nq, H, D] and the float32 row log-sum-exp [B, H, Nq] of
    softmax(q k^T * scale) v, for `flash_attn_backward`."""
    b, nq, h, d, nk, hk = _check(q, k, v, k_lens)
    scale = d ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not (b and nq and h and d and nk):
        dt = torch.float64 if q.dtype == torch.float64 else torch.float32
        return (torch.zeros_like(q, memory_format=torch.contiguous_format),
                torch.full((b, h, nq), -math.inf, device=q.device, dtype=dt))
    if not _kernel_ok(q, d, scale):
        _fallback("flash_attn_lse", q, k, v)
        return _torch_lse(q, k, v, scale, causal, k_lens)
    q, qs = heads_layout(q, _MOST)
    k, ks = heads_layout(k, _MOST)
    v, vs = heads_layout(v, _MOST)
    lens = _lens32(k_lens, nk)
    out = fresh(q)
    lse = q.new_empty((b, h, nq), dtype=torch.float32)
    size = bytes_on(q, "oga_attention_lse_workspace_bytes", b, nq, nk, h, hk, d, bool(causal))
    ws = scratch(q, size) if size else None
    _hip("flash_attn_lse")
    call_on(q, "oga_attention_lse", q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, out.data_ptr(),
            (nq * h * d, h * d, d), lse.data_ptr(), b, nq, nk, h, hk, d, scale, bool(causal),
            None if lens is None else lens.data_ptr(), None if ws is None else ws.data_ptr(), size)
    return out, lse


def flash_attn_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                        lse: torch.Tensor, softmax_scale: float | None = None, causal: bool = False,
                        k_lens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """dq, dk, dv of the call of `flash_attn_lse` that gave `out` and `lse`
    with these arguments. Deterministic: no sum goes through atomics."""
    b, nq, h, d, nk, hk = _check(q, k, v, k_lens)
    _check_grad(dout, q, out, lse)
    scale = d ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not (b and nq and h and d and nk):
        return tuple(torch.zeros_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
    if not _kernel_ok(q, d, scale) or lse.dtype != torch.float32:
        _fallback("flash_attn_backward", q, k, v)
        return _torch_backward(dout, q, k, v, lse, scale, causal, k_lens)
    q, qs = heads_layout(q, _MOST)
    k, ks = heads_layout(k, _MOST)
    v, vs = heads_layout(v, _MOST)
    out, os = heads_layout(out, _MOST)
    dout, ds = heads_layout(dout, _MOST)
    if not lse.is_contiguous():
        lse = lse.contiguous()
    lens = _lens32(k_lens, nk)
    dq, dk, dv = fresh(q), fresh(k), fresh(v)
    dqs, dks = (nq * h * d, h * d, d), (nk * hk * d, hk * d, d)
    size = bytes_on(q, "oga_attention_bwd_workspace_bytes", b, nq, nk, h, hk, d, bool(causal))
    ws = scratch(q, size)
    _hip("flash_attn_backward")
    call_on(q, "oga_attention_bwd", dout.data_ptr(), ds, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
            out.data_ptr(), os, lse.data_ptr(), dq.data_ptr(), dqs, dk.data_ptr(), dks, dv.data_ptr(), dks, b, nq, nk,
            h, hk, d, scale, bool(causal), None if lens is None else lens.data_ptr(), ws.data_ptr(), size)
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, softmax_scale, causal, k_lens):
        out, lse = flash_attn_lse(q, k, v, softmax_scale, causal, k_lens)
        ctx.save_for_backward(q, k, v, out, lse, k_lens)
        ctx.how = softmax_scale, causal
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, k_lens = ctx.saved_tensors
        return (*flash_attn_backward(dout, q, k, v, out, lse, *ctx.how, k_lens), None, None, None)


def attention_with_grad(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, softmax_scale: float | None = None,
                        causal: bool = False, k_lens: torch.Tensor | None = None) -> torch.Tensor:
    """`flash_attn_lse`'s output, differentiable in q, k and v."""
    return _Attention.apply(q, k, v, softmax_scale, causal, k_lens)
