"""Head norms with the position rotation (opengenie_amd.head_rope) against
their formulas in float64.

Bounds: results are rounded once, by at most u = eps / 2 of the type (fp16
also by half its subnormal step). The float32 chain has under 30 roundings of
values no larger than the terms summed, 2^-19 of their absolute sum; the
reciprocal root of a mean of up to 256 squares is off by under 2^-16
relatively. A weight's gradient sums over rows, in float32 runs of under 2^6
terms a lane and less than 2^8 partial sums: 2^-15 of the absolute sum.
"""

from __future__ import annotations

import pytest
import torch

from opengenie_amd import _lib
from opengenie_amd import head_rope as H
from opengenie_amd import ltx_ops as L
from opengenie_amd.rope import rotary_cos_sin

from helpers import gen

EPS = 1e-6


def rnd(*shape, seed, dtype=torch.float32, device="cpu", std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen(seed)) * std + mean).to(dtype).to(device)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def turn64(x, cos, sin, layout, absolute=False):
    """Rot in float64, or the absolute sum of its terms."""
    half = cos.shape[-1]
    i = torch.arange(half, device=x.device)
    one, two = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
    y = x.abs().clone() if absolute else x.clone()
    a, b = x[..., one], x[..., two]
    if absolute:
        y[..., one] = (a * cos).abs() + (b * sin).abs()
        y[..., two] = (b * cos).abs() + (a * sin).abs()
    else:
        y[..., one] = a * cos - b * sin
        y[..., two] = b * cos + a * sin
    return y


def tables64(cos, sin, n, positions):
    if positions is None:
        return cos[:n].double()[None, :, None], sin[:n].double()[None, :, None]
    at = positions.long().clamp(0, cos.shape[0] - 1)
    return cos.double()[at][:, :, None], sin.double()[at][:, :, None]


def close(got, want, terms, dtype, rel, what):
    bound = rel * terms + half_step(dtype) * (want.abs() + rel * terms) * 1.001
    bound = bound + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
    off = ((got.double() - want).abs() - bound).max().item()
    assert off <= 0, f"{what}: {off:.3g} over the bound"


def check(q, k, qw, kw, cos, sin, layout, positions, grads=True):
    q_out, k_out = H.qk_head_rmsnorm_rope(q, k, qw, kw, EPS, cos, sin, layout=layout, positions=positions)
    c, s = tables64(cos, sin, q.shape[1], positions)
    dq_out, dk_out = (rnd(*t.shape, seed=90 + i, dtype=t.dtype, device=t.device) for i, t in enumerate((q, k)))
    back = H.qk_head_rmsnorm_rope_backward(dq_out, dk_out, q, k, qw, kw, EPS, cos, sin, layout=layout,
                                           positions=positions)
    for x, w, y, dy, dx, dw, name in ((q, qw, q_out, dq_out, back[0], back[2], "q"),
                                      (k, kw, k_out, dk_out, back[1], back[3], "k")):
        x64 = x.double()
        w64 = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
        r = 1 / torch.sqrt(x64.square().mean(-1, keepdim=True) + EPS)
        n = x64 * r
        close(y, turn64(n * w64, c, s, layout), turn64(n * w64, c, s, layout, True), x.dtype, 2.0 ** -15, name)
        dn, an = turn64(dy.double(), c, -s, layout), turn64(dy.double(), c, s, layout, True)
        along = (dn * w64 * n).mean(-1, keepdim=True)
        terms = r * ((an * w64).abs() + n.abs() * (an * w64 * n).abs().mean(-1, keepdim=True))
        close(dx, r * (dn * w64 - n * along), terms, x.dtype, 2.0 ** -14, "d" + name)
        if w is None:
            assert dw is None
        else:
            assert dw.dtype == w.dtype
            close(dw, (dn * n).sum((0, 1, 2)), (an * n.abs()).sum((0, 1, 2)), w.dtype, 2.0 ** -15, f"d{name}w")
    return (q_out, k_out, *back)


# ------------------------------------------------------------------- CPU
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 48), (40, 24)])
def test_torch_path_is_the_formulas(dim, rot, layout):
    q, k = rnd(2, 7, 3, dim, seed=1, dtype=torch.bfloat16), rnd(2, 7, 1, dim, seed=2, dtype=torch.bfloat16)
    cos, sin = rotary_cos_sin(20, rot)
    pos = torch.randint(0, 20, (2, 7), generator=gen(3))
    check(q, k, rnd(dim, seed=4, mean=1.0), None, cos, sin, layout, pos)
    check(q, k, None, rnd(dim, seed=5, dtype=torch.bfloat16), cos, sin, layout, None)
    x = rnd(2, 7, 3, dim, seed=6)
    turned = H.apply_rope(x, cos, sin, layout=layout)
    torch.testing.assert_close(H.apply_rope(turned, cos, sin, layout=layout, inverse=True), x, rtol=1e-5, atol=1e-5)
    assert torch.equal(turned[..., rot:], x[..., rot:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradients_against_differences(layout):
    q, k = rnd(2, 3, 2, 8, seed=7).double(), rnd(2, 3, 1, 8, seed=8).double()
    qw, kw = rnd(8, seed=9, mean=1.0).double(), rnd(8, seed=10, mean=1.0).double()
    cos, sin = rotary_cos_sin(3, 6, dtype=torch.float64)
    for t in (q, k, qw, kw):
        t.requires_grad_(True)
    assert torch.autograd.gradcheck(
        lambda *t: H.qk_head_rmsnorm_rope_with_grad(*t, EPS, cos, sin, layout=layout), (q, k, qw, kw))


def test_tables():
    """Angles of each kind of table against its formula."""
    cos, sin = rotary_cos_sin(100, 16, theta=100.0, dtype=torch.float64)
    freq = 100.0 ** (-torch.arange(8, dtype=torch.float64) / 8)
    ang = torch.arange(100, dtype=torch.float64)[:, None] * freq
    torch.testing.assert_close(cos, ang.cos(), rtol=0, atol=1e-12)
    torch.testing.assert_close(sin, ang.sin(), rtol=0, atol=1e-12)
    cos, _ = rotary_cos_sin(100, 16, theta=100.0, scaling="linear", factor=4.0, dtype=torch.float64)
    torch.testing.assert_close(cos, (ang / 4).cos(), rtol=0, atol=1e-12)
    cos, _ = rotary_cos_sin(100, 16, theta=100.0, scaling="ntk", factor=4.0, dtype=torch.float64)
    low = (100.0 * 4.0 ** (16 / 14)) ** (-torch.arange(8, dtype=torch.float64) / 8)
    torch.testing.assert_close(cos, (torch.arange(100, dtype=torch.float64)[:, None] * low).cos(), rtol=0, atol=1e-12)
    # the slowest plane of the base-stretched table turns `factor` times slower
    assert abs(low[-1] * 4.0 / freq[-1] - 1) < 1e-12
    cos, sin = rotary_cos_sin(64, 16, theta=100.0, scaling="ramp", factor=4.0, original_length=32, fast=4.0, slow=1.0,
                              dtype=torch.float64)
    turns = 32 * freq / (2 * torch.pi)
    keep = ((turns - 1.0) / 3.0).clamp(0, 1)
    ramp = torch.arange(64, dtype=torch.float64)[:, None] * (freq * keep + freq / 4 * (1 - keep))
    torch.testing.assert_close(sin, ramp.sin(), rtol=0, atol=1e-12)
    far, _ = rotary_cos_sin(3, 16, start=10 ** 9, dtype=torch.float64)
    assert abs(far[2, 0].item() - torch.tensor(1e9 + 2, dtype=torch.float64).cos().item()) < 1e-12
    for kw in ({"rotary_dim": 7}, {"rotary_dim": 16, "scaling": "other"}, {"rotary_dim": 16, "factor": 2.0},
               {"rotary_dim": 16, "scaling": "ramp", "factor": 2.0}):
        with pytest.raises(ValueError):
            rotary_cos_sin(4, **kw)


def test_empty_inputs():
    cos, sin = rotary_cos_sin(4, 16)
    q, k, w = rnd(2, 0, 3, 64, seed=1), rnd(2, 0, 1, 64, seed=1), rnd(64, seed=2)
    a, b = H.qk_head_rmsnorm_rope(q, k, w, w, EPS, cos, sin)
    assert a.shape == q.shape and b.shape == k.shape
    _, _, dqw, dkw = H.qk_head_rmsnorm_rope_backward(q, k, q, k, w, w, EPS, cos, sin)
    assert not dqw.any() and not dkw.any()
    assert H.apply_rope(q, cos, sin).shape == q.shape


def test_refusals():
    cos, sin = rotary_cos_sin(9, 32)
    q, k, w = rnd(2, 9, 4, 64, seed=1), rnd(2, 9, 2, 64, seed=2), rnd(64, seed=3)
    pos = torch.zeros((2, 9), dtype=torch.int32)
    ok = dict(q=q, k=k, q_weight=w, k_weight=w, eps=EPS, cos=cos, sin=sin, layout="half", positions=pos)
    H.qk_head_rmsnorm_rope(**ok)
    for bad in ({"layout": "neox"}, {"q": q[0]}, {"k": k[:, :3]}, {"k": k.double()}, {"k": k[..., :32]},
                {"cos": cos[None]}, {"sin": sin[:, :8]}, {"sin": sin.double()}, {"positions": pos[:, :3]},
                {"positions": pos.float()}, {"q_weight": w[:32]}, {"k_weight": w.int()},
                {"positions": None, "cos": cos[:8], "sin": sin[:8]}, {"cos": torch.ones(9, 33), "sin": torch.ones(9, 33)},
                {"cos": cos[:0], "sin": sin[:0]}):
        with pytest.raises(ValueError):
            H.qk_head_rmsnorm_rope(**{**ok, **bad})
    with pytest.raises(ValueError):
        H.qk_head_rmsnorm_rope_backward(q[:1], k, q, k, w, w, EPS, cos, sin)
    with pytest.raises(ValueError):
        H.qk_head_rmsnorm_rope_backward(q, k.double(), q, k, w, w, EPS, cos, sin)


@pytest.mark.skipif(not _lib.available(), reason="library not built")
def test_entry_points_refuse_what_the_kernels_do_not_take():
    """Nothing is launched: every call here fails its argument checks."""
    lib = _lib.load()
    st, pst, p = _lib.strides((8192, 512, 128)), _lib.strides((8, 1)), 4096

    def fwd(dt=0, q=p, qs=st, k=p, w=p, wdt=0, cos=p, cdt=1, cs=64, length=8, pos=None, batch=1, tokens=8, heads=4,
            kv=1, dim=128, rot=128):
        return lib.oga_head_rmsnorm_rope(dt, q, qs, k, st, w, w, wdt, cos, p, cdt, cs, length, pos, 0, pst, p, st, p,
                                         st, batch, tokens, heads, kv, dim, rot, 0, 0, 1, 1e-6, None)

    for kw in ({"dt": 1}, {"dt": 7}, {"wdt": 2}, {"cdt": 2}, {"q": None}, {"q": 4100}, {"k": None},
               {"qs": _lib.strides((8192, 512, 4))}, {"w": 4104}, {"cos": None}, {"cos": 4104}, {"cs": 6}, {"cs": -64},
               {"length": 7}, {"length": 0, "pos": p}, {"batch": 0}, {"tokens": 0}, {"heads": 0}, {"kv": -1},
               {"rot": 8}, {"rot": 144}, {"rot": 24}):
        assert fwd(**kw) == -1, kw
    assert fwd(dim=96, rot=96) == -2 and fwd(batch=1 << 20, tokens=1 << 12, length=1 << 12) == -2
    need = lib.oga_head_rmsnorm_rope_bwd_workspace_bytes(128)
    assert need > 0 and lib.oga_head_rmsnorm_rope_bwd_workspace_bytes(96) == 0

    def bwd(ws, size, dqw=p, qw=p):
        return lib.oga_head_rmsnorm_rope_bwd(0, p, st, p, st, p, st, p, st, qw, p, 0, p, p, 1, 64, 8, None, 0, pst, p,
                                             st, p, st, dqw, None, 1, 8, 4, 1, 128, 128, 0, 1e-6, ws, size, None)

    assert bwd(None, need) == -1 and bwd(p, need - 1) == -1 and bwd(p, need, qw=None) == -1


# ------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(64, 64), (64, 16), (64, 48), (128, 128), (128, 96), (128, 80), (256, 256),
                                     (256, 176), (256, 16)])
def test_gpu_against_float64(dim, rot, layout, monkeypatch):
    monkeypatch.setenv("OPENGENIE_AMD_STRICT", "1")
    L.reset_hip_calls()
    for i, (b, n, h, hk, dt, tdt, wdt) in enumerate([
            (1, 1, 1, 1, torch.bfloat16, torch.float32, torch.float32),
            (3, 37, 5, 2, torch.bfloat16, torch.bfloat16, torch.bfloat16),
            (2, 131, 32, 8, torch.float16, torch.float32, torch.float32),
            (1, 259, 9, 9, torch.bfloat16, torch.float32, None)]):
        q, k = rnd(b, n, h, dim, seed=20 + i, dtype=dt, device="cuda"), rnd(b, n, hk, dim, seed=30 + i, dtype=dt, device="cuda")
        qw, kw = (None if wdt is None else rnd(dim, seed=40 + i + j, dtype=wdt, device="cuda", mean=1.0, std=0.2)
                  for j in range(2))
        cos, sin = rotary_cos_sin(3 * n, rot, device="cuda", dtype=tdt)
        check(q, k, qw, kw, cos, sin, layout, None)
        for pdt in (torch.int32, torch.int64):
            pos = torch.randint(-3, 3 * n + 5, (b, n), generator=gen(50 + i)).to(pdt).cuda()
            check(q, k, qw, kw, cos, sin, layout, pos)
        x64 = q.double()
        c, s = tables64(cos, sin, n, pos)
        for inverse in (False, True):
            y = H.apply_rope(q, cos, sin, layout=layout, positions=pos, inverse=inverse)
            sg = -s if inverse else s
            close(y, turn64(x64, c, sg, layout), turn64(x64, c, s, layout, True), dt, 2.0 ** -21, "rope")
            assert torch.equal(y[..., rot:], q[..., rot:])
    assert set(L.collect_hip_calls()) == {"qk_head_rmsnorm_rope", "qk_head_rmsnorm_rope_backward", "apply_rope"}


@pytest.mark.gpu
def test_gpu_layouts_give_the_same_bits():
    """Views of a packed projection, expanded gradients, odd offsets, sliced
    tables and mixed weight dtypes against contiguous inputs."""
    b, n, h, d = 2, 33, 4, 128
    qkv = rnd(b, n, 3, h, d, seed=60, dtype=torch.bfloat16, device="cuda")
    q, k, _ = qkv.unbind(2)
    w = rnd(d, seed=61, device="cuda", mean=1.0).to(torch.bfloat16)
    cos, sin = rotary_cos_sin(2 * n, d, device="cuda")
    wide = torch.cat((cos, sin), 1)
    pos = torch.randint(0, 2 * n, (n, b), generator=gen(62)).cuda().t()
    dy = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(b, n, h, d)
    want = H.qk_head_rmsnorm_rope(q.contiguous(), k.contiguous(), w, w, EPS, cos, sin, positions=pos.contiguous())
    got = H.qk_head_rmsnorm_rope(q, k, w, w, EPS, wide[:, :d // 2], wide[:, d // 2:], positions=pos)
    odd = torch.empty(q.numel() + 1, device="cuda", dtype=q.dtype)[1:].view(q.shape).copy_(q)
    got2 = H.qk_head_rmsnorm_rope(odd, k, w, w.float(), EPS, cos, sin, positions=pos)
    for x, y, z in zip(want, got, got2):
        assert torch.equal(x, y) and torch.equal(x, z)
    a = H.qk_head_rmsnorm_rope_backward(dy, dy, q, k, w, w, EPS, cos, sin, positions=pos)
    c = H.qk_head_rmsnorm_rope_backward(dy.contiguous(), dy.contiguous(), q.contiguous(), k.contiguous(), w, w, EPS,
                                        cos, sin, positions=pos)
    for x, y in zip(a, c):
        assert torch.equal(x, y)
    mixed = H.qk_head_rmsnorm_rope_backward(dy, dy, q, k, w, w.float(), EPS, cos, sin, positions=pos)
    assert mixed[2].dtype == torch.bfloat16 and mixed[3].dtype == torch.float32
    assert torch.equal(mixed[2], a[2]) and torch.equal(mixed[3].to(torch.bfloat16), a[3])


@pytest.mark.gpu
def test_gpu_special_values_stay_in_their_head():
    q = rnd(1, 9, 4, 64, seed=70, dtype=torch.bfloat16, device="cuda")
    k = rnd(1, 9, 4, 64, seed=71, dtype=torch.bfloat16, device="cuda")
    cos, sin = rotary_cos_sin(9, 32, device="cuda")
    want = H.qk_head_rmsnorm_rope(q, k, None, None, EPS, cos, sin)[0]
    q2 = q.clone()
    q2[0, 3, 1, 5], q2[0, 4, 2, 40] = float("nan"), float("inf")
    q2[0, 5, 3] = 0.0
    got = H.qk_head_rmsnorm_rope(q2, k, None, None, EPS, cos, sin)[0]
    for n, h in ((3, 1), (4, 2)):
        assert torch.isnan(got[0, n, h]).any()
    assert not got[0, 5, 3].any()
    for n, h in ((3, 1), (4, 2), (5, 3)):
        got[0, n, h] = want[0, n, h]
    assert torch.equal(got, want)
    # an infinity that is not turned stays alone
    x = q.clone()
    x[0, 2, 0, 63] = float("inf")
    y = H.apply_rope(x, cos, sin)
    assert torch.isfinite(y).sum() == y.numel() - 1 and torch.isinf(y[0, 2, 0, 63])


@pytest.mark.gpu
def test_gpu_same_bits_twice_in_a_graph_and_on_another_stream():
    q = rnd(2, 700, 8, 128, seed=80, dtype=torch.bfloat16, device="cuda")
    k = rnd(2, 700, 2, 128, seed=81, dtype=torch.bfloat16, device="cuda")
    w = rnd(128, seed=82, device="cuda", mean=1.0)
    cos, sin = rotary_cos_sin(700, 128, device="cuda")

    def step(q, k):
        y = H.qk_head_rmsnorm_rope(q, k, w, w, EPS, cos, sin)
        return (*y, *H.qk_head_rmsnorm_rope_backward(*y, q, k, w, w, EPS, cos, sin))

    want = step(q, k)
    for x, y in zip(want, step(q, k)):
        assert torch.equal(x, y)
    other = step(k.repeat(1, 1, 4, 1), q[:, :, :2])
    static = [q.clone(), k.clone()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for x, y in zip(want, step(*static)):
            assert torch.equal(x, y)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*static)
    for fresh, expect in (((k.repeat(1, 1, 4, 1), q[:, :, :2]), other), ((q, k), want)) * 2:
        for s, t in zip(static, fresh):
            s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        step(q, k)
        for x, y in zip(got, expect):
            assert torch.equal(x, y)
