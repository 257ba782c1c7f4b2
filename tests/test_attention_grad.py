"""Attention with gradients (opengenie_amd.attention_grad) against its formulas
in float64.

Bounds: a rounding to bf16 is off by at most u = 2^-8 of the value. P and dS
are rounded once before the second products, results once, so out is off by at
most u (sum P |v| + |out|), and Delta, summed from the rounded out, by that
against |dout|. A float32 dot product of D terms is off by (D + 2) 2^-24 of
its terms' absolute sum, which is a relative error of P (twice: in its own
score and in the row's lse, with 2^-20 for the exponential and logarithm).
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from opengenie_amd import _lib
from opengenie_amd import attention_grad as G
from opengenie_amd import ltx_ops as L

from helpers import gen

U = 2.0 ** -8
F32 = 2.0 ** -24


def inputs(b, nq, nk, h, hk, d, seed, device="cpu", std=1.0, dtype=torch.bfloat16):
    g = gen(seed)

    def t(n, heads):
        return (torch.randn((b, n, heads, d), generator=g) * std).to(dtype).to(device)

    return t(nq, h), t(nk, hk), t(nk, hk), t(nq, h)


def exact(q, k, v, dout, scale, causal, lens):
    """Results in float64 and the bounds of the kernels' errors, per output."""
    b, nq, h, d = q.shape
    nk, hk = k.shape[1], k.shape[2]
    r = {n: torch.zeros(t.shape, dtype=torch.float64, device=q.device) for n, t in
         (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    e = {n: torch.zeros_like(t) for n, t in r.items()}
    r["lse"] = torch.full((b, h, nq), -math.inf, dtype=torch.float64, device=q.device)
    e["lse"] = torch.zeros_like(r["lse"])
    for i in range(b):
        n = nk if lens is None else min(max(int(lens[i]), 0), nk)
        for j in range(h):
            c = j // (h // hk)
            x, kk, vv, do = (t.double() for t in (q[i, :, j], k[i, :n, c], v[i, :n, c], dout[i, :, j]))
            s = x @ kk.t() * scale
            if causal:
                hide = torch.arange(n, device=q.device) > torch.arange(nq, device=q.device)[:, None] + n - nq
                s = s.masked_fill(hide, -math.inf)
            some = (s > -math.inf).any(1) if n else torch.zeros(nq, dtype=torch.bool, device=q.device)
            if not some.any():
                continue
            x, do, s = x[some], do[some], s[some]
            z = torch.logsumexp(s, 1)
            p = torch.exp(s - z[:, None])
            es = (d + 2) * F32 * scale * (x.abs() @ kk.abs().t())
            es = es.masked_fill(s == -math.inf, 0.0).amax(1, keepdim=True)
            rel = 2 * es + 2.0 ** -20  # of P before its rounding
            o = p @ vv
            eo = (U + rel) * (p @ vv.abs()) * 1.01
            dp = do @ vv.t()
            delta = (do * o).sum(1, keepdim=True)
            # out is rounded once more before Delta is summed from it
            ed = (do.abs() * (eo + U * (o.abs() + eo))).sum(1, keepdim=True) + (d + 2) * F32 * (do * o).abs().sum(1, keepdim=True)
            ds = p * (dp - delta)
            eds = (U + rel) * ds.abs() * 1.01 + p * (ed + (d + 2) * F32 * (do.abs() @ vv.abs().t())) * 1.01
            r["lse"][i, j, some], e["lse"][i, j, some] = z, es[:, 0] + 2.0 ** -20 * (1 + z.abs())
            r["out"][i, some, j], e["out"][i, some, j] = o, eo
            r["dq"][i, some, j], e["dq"][i, some, j] = scale * (ds @ kk), scale * (eds @ kk.abs())
            r["dk"][i, :n, c] += scale * (ds.t() @ x)
            e["dk"][i, :n, c] += scale * (eds.t() @ x.abs())
            r["dv"][i, :n, c] += p.t() @ do
            e["dv"][i, :n, c] += (U + rel[:, 0].max()) * (p.t() @ do.abs()) * 1.01
    for n in ("out", "dq", "dk", "dv"):  # the sums themselves, then the rounding of the result
        e[n] = e[n] * 1.01 + U * (r[n].abs() + e[n]) + 1e-30
    return r, e


def check(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    assert torch.isfinite(got[~inf]).all(), what
    off = (got - want).abs()[~inf] - bound[~inf]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: {off.max().item():.3g} over the bound"


def run_and_check(q, k, v, dout, scale=None, causal=False, lens=None, k_lens=None):
    f = q.shape[-1] ** -0.5 if scale is None else scale
    out, lse = G.flash_attn_lse(q, k, v, scale, causal, k_lens)
    grads = G.flash_attn_backward(dout, q, k, v, out, lse, scale, causal, k_lens)
    r, e = exact(q, k, v, dout, f, causal, lens)
    for name, t in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        check(t, r[name], e[name], name)
    return out, lse, grads


# ------------------------------------------------------------------- CPU
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", [(1, 1, 1, 2, 1, 64), (2, 9, 13, 4, 2, 64), (2, 13, 9, 2, 2, 128)])
def test_torch_path_is_the_formulas(shape, causal):
    q, k, v, dout = inputs(*shape, seed=1)
    lens = [max(shape[2] - 4, 0), shape[2]][: shape[0]]
    k_lens = torch.tensor(lens, dtype=torch.int64)
    run_and_check(q, k, v, dout, causal=causal, lens=lens, k_lens=k_lens)


@pytest.mark.parametrize("causal", [False, True])
def test_gradients_against_differences(causal):
    q, k, v, _ = inputs(2, 3, 5, 2, 1, 8, seed=2, dtype=torch.float64)
    lens = torch.tensor([5, 2], dtype=torch.int32)
    for t in (q, k, v):
        t.requires_grad_(True)
    assert torch.autograd.gradcheck(lambda *t: G.attention_with_grad(*t, None, causal, lens), (q, k, v))


def test_rows_without_a_key_and_unread_padding():
    q, k, v, dout = inputs(2, 6, 4, 2, 2, 64, seed=3)
    k[0, 2:], v[0, 2:] = math.nan, math.inf
    k[1], v[1] = math.nan, math.nan
    k_lens = torch.tensor([2, 0], dtype=torch.int32)
    out, lse, (dq, dk, dv) = run_and_check(q, k, v, dout, causal=True, lens=[2, 0], k_lens=k_lens)
    assert not out[1].any() and not dq[1].any() and not dk[1].any() and not dv[1].any()
    assert not out[0, :4].any() and (lse[0, :, :4] == -math.inf).all() and (lse[1] == -math.inf).all()


def test_empty_inputs():
    q, k, v, dout = inputs(2, 3, 0, 2, 2, 64, seed=4)
    out, lse = G.flash_attn_lse(q, k, v)
    assert not out.any() and (lse == -math.inf).all()
    dq, dk, dv = G.flash_attn_backward(dout, q, k, v, out, lse)
    assert not dq.any() and dk.shape == k.shape and dv.shape == v.shape
    q, k, v, dout = inputs(2, 0, 3, 2, 2, 64, seed=4)
    out, lse = G.flash_attn_lse(q, k, v)
    dq, dk, dv = G.flash_attn_backward(dout, q, k, v, out, lse)
    assert out.shape == q.shape and lse.shape == (2, 2, 0) and not dk.any() and not dv.any()


def test_refusals():
    q, k, v, dout = inputs(2, 5, 7, 4, 2, 64, seed=5)
    out, lse = G.flash_attn_lse(q, k, v)
    bad = [(q[0], k, v), (q, k[:1], v[:1]), (q, k, v[:, :3]), (q[:, :, :3], k, v), (q, k[..., :32], v[..., :32]),
           (q.float(), k, v), (q.int(), k.int(), v.int()), (q, k[:, :, :0], v[:, :, :0])]
    for args in bad:
        with pytest.raises(ValueError):
            G.flash_attn_lse(*args)
    for k_lens in (torch.tensor([1, 2, 3]), torch.tensor([1.0, 2.0]), torch.tensor([[1], [2]])):
        with pytest.raises(ValueError):
            G.flash_attn_lse(q, k, v, k_lens=k_lens)
    for d, o, s in ((dout[:, :3], out, lse), (dout, out[:1], lse), (dout, out, lse[:, :, :2]), (dout.float(), out, lse)):
        with pytest.raises(ValueError):
            G.flash_attn_backward(d, q, k, v, o, s)


@pytest.mark.skipif(not _lib.available(), reason="library not built")
def test_entry_points_refuse_what_the_kernels_do_not_take():
    """Nothing is launched: every call here fails its argument checks."""
    lib = _lib.load()
    st, p = _lib.strides((8192, 128, 128)), 4096

    def lse(q=p, qs=st, batch=1, nq=4, nk=4, heads=1, kv_heads=1, dim=128, scale=0.1,
            ws=None, size=0):
        return lib.oga_attention_lse(q, qs, p, st, p, st, p, st, p, batch, nq, nk, heads, kv_heads, dim, scale, 0,
                                     None, ws, size, None)

    assert lse(dim=96) == -2 and lse(dim=32) == -2
    for kw in ({"q": None}, {"q": 4104}, {"qs": _lib.strides((8192, 4, 128))}, {"qs": _lib.strides((0, 1 << 24, 8))},
               {"batch": 0}, {"nq": 0}, {"nk": 0}, {"heads": 3, "kv_heads": 2}, {"scale": 0.0},
               {"scale": float("nan")}, {"scale": float("inf")}):
        assert lse(**kw) == -1, kw
    assert lse(nq=1 << 31) == -2 and lse(batch=1 << 20, heads=1 << 20) == -2
    assert lse(batch=1 << 19, heads=32) == -2 and lse(batch=1 << 19, nq=8, nk=4096) == -2  # grids past 2^32 threads
    need = lib.oga_attention_lse_workspace_bytes(1, 4, 4096, 1, 1, 128, 0)
    assert need > 0  # one block, cut over its keys
    for kw in ({}, {"ws": p, "size": need - 1}, {"ws": p + 16, "size": need}):
        assert lse(nk=4096, **kw) == -1 and b"workspace" in lib.oga_last_error()
    assert lse(nq=1, heads=4, qs=_lib.strides((0, 0, 1 << 24))) == -1  # one query: heads are its rows
    need = lib.oga_attention_bwd_workspace_bytes(1, 4, 4, 1, 1, 128, 0)
    assert need >= 512 and lib.oga_attention_bwd_workspace_bytes(1, 4, 4, 3, 2, 128, 0) == 0

    def bwd(ws, size):
        return lib.oga_attention_bwd(p, st, p, st, p, st, p, st, p, st, p, p, st, p, st, p, st, 1, 4, 4, 1, 1, 128,
                                     0.1, 0, None, ws, size, None)

    assert bwd(None, need) == -1 and bwd(p, need - 1) == -1 and bwd(p + 16, need) == -1
    assert b"workspace" in lib.oga_last_error()


# ------------------------------------------------------------------- GPU
SHAPES = [
    (1, 1, 1, 1, 1, 128), (1, 1, 1, 1, 1, 64), (3, 1, 70, 4, 2, 128), (2, 64, 64, 2, 2, 128), (1, 65, 63, 2, 1, 64),
    (2, 33, 257, 4, 1, 128), (1, 257, 255, 2, 2, 64), (1, 300, 129, 3, 3, 128), (2, 190, 321, 6, 2, 64),
    (1, 513, 700, 2, 2, 128), (1, 1030, 77, 2, 1, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gpu_against_float64(shape, causal, monkeypatch):
    monkeypatch.setenv("OPENGENIE_AMD_STRICT", "1")
    q, k, v, dout = inputs(*shape, seed=11, device="cuda")
    L.reset_hip_calls()
    run_and_check(q, k, v, dout, causal=causal)
    assert L.collect_hip_calls() == {"flash_attn_lse": 1, "flash_attn_backward": 1}


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_gpu_padded_batch(dim, causal):
    """Lengths of nothing, one key, an end inside a tile, a tile's end and
    beyond; what lies behind them is infinite or not a number."""
    lens = [0, 1, 61, 128, 200, 999]
    q, k, v, dout = inputs(6, 150, 200, 4, 2, dim, seed=12, device="cuda")
    for i, n in enumerate(lens):
        k[i, n:], v[i, n:] = math.nan, math.inf
    for dt in (torch.int32, torch.int64):
        k_lens = torch.tensor(lens, device="cuda", dtype=dt)
        out, lse, (dq, dk, dv) = run_and_check(q, k, v, dout, causal=causal, lens=lens, k_lens=k_lens)
    assert not out[0].any() and not dk[0].any() and not dk[1, 1:].any() and not dv[2, 61:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_gpu_large_and_small_scores(dim):
    """Scores of hundreds (one key takes a row), and scores whose running
    maximum rises over the keys; a scale of the caller's own."""
    q, k, v, dout = inputs(1, 130, 400, 2, 2, dim, seed=13, device="cuda", std=4.0)
    run_and_check(q, k, v, dout, scale=0.5)
    k = (k.float() * torch.linspace(0.01, 1.5, 400, device="cuda")[None, :, None, None]).to(torch.bfloat16)
    run_and_check(q, k, v, dout)
    run_and_check(q, k, v, dout, scale=1e-4, causal=True)


@pytest.mark.gpu
def test_gpu_layouts_give_the_same_bits():
    """Views of a packed projection, an expanded gradient, transposed and
    misaligned inputs against contiguous ones."""
    b, n, h, d = 2, 97, 3, 128
    qkv = torch.randn((b, n, 3, h, d), generator=gen(14)).to(torch.bfloat16).cuda()
    q, k, v = qkv.unbind(2)
    dout = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(b, n, h, d)
    c = [t.contiguous() for t in (q, k, v)]
    out, lse = G.flash_attn_lse(*c)
    grads = G.flash_attn_backward(dout.contiguous(), *c, out, lse)
    out2, lse2 = G.flash_attn_lse(q, k, v)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    out2 = out2.transpose(1, 2).contiguous().transpose(1, 2)
    for x, y in zip(grads, G.flash_attn_backward(dout, q, k, v, out2, lse2)):
        assert torch.equal(x, y)
    odd = []
    for t in c:
        flat = torch.empty(t.numel() + 3, device="cuda", dtype=torch.bfloat16)
        odd.append(flat[3:].view(t.shape).copy_(t))
    assert torch.equal(G.flash_attn_lse(*odd)[0], out)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 700, 130, 4, 2, 128), (2, 300, 300, 4, 4, 64)], ids=str)
def test_gpu_same_bits_twice_and_in_a_graph(shape):
    """Two calls, and replays of a captured pair of calls between eager work
    on other inputs, give the same bits as the first eager call."""
    q, k, v, dout = inputs(*shape, seed=15, device="cuda")
    k_lens = torch.tensor([shape[2] - 3] * shape[0], device="cuda", dtype=torch.int32)

    def step(q, k, v, dout):
        out, lse = G.flash_attn_lse(q, k, v, causal=True, k_lens=k_lens)
        return (out, lse, *G.flash_attn_backward(dout, q, k, v, out, lse, causal=True, k_lens=k_lens))

    want = step(q, k, v, dout)
    for x, y in zip(want, step(q, k, v, dout)):
        assert torch.equal(x, y)
    other = inputs(*shape, seed=16, device="cuda")
    static = [t.clone() for t in (q, k, v, dout)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*static)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*static)
    for fresh, expect in ((other, None), ((q, k, v, dout), want), (other, None), ((q, k, v, dout), want)):
        for s, t in zip(static, fresh):
            s.copy_(t)
        expect = expect if expect is not None else step(*other)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, expect):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_gpu_autograd_on_another_stream():
    q, k, v, dout = inputs(1, 200, 100, 4, 2, 64, seed=17, device="cuda")
    out, lse = G.flash_attn_lse(q, k, v)
    want = G.flash_attn_backward(dout, q, k, v, out, lse)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        G.attention_with_grad(*leaves).backward(dout)
    stream.synchronize()
    for t, w in zip(leaves, want):
        assert torch.equal(t.grad, w)


@pytest.mark.gpu
def test_gpu_strict_mode_refuses_what_falls_back(monkeypatch):
    q, k, v, dout = inputs(1, 5, 6, 2, 2, 32, seed=18, device="cuda")
    out, lse, _ = run_and_check(q, k, v, dout)
    monkeypatch.setenv("OPENGENIE_AMD_STRICT", "1")
    with pytest.raises(RuntimeError):
        G.flash_attn_lse(q, k, v)
    with pytest.raises(RuntimeError):
        G.flash_attn_backward(dout, q, k, v, out, lse)
    with pytest.raises(ValueError):
        G.flash_attn_lse(q, k.cpu(), v.cpu())
