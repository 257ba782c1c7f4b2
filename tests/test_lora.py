"""Low-rank adapters (opengenie_amd.lora) against their formulas in float64.

Bounds: results are rounded once, by at most u = eps / 2 of the type (fp16
also by half its subnormal step). A float32 sum of n terms is off by n 2^-24 of
their absolute sum. low and dlow enter the second products as two 16-bit halves
(bf16: what is left is 2^-16 of the value; fp16: 2^-22 and 2^-25 absolutely),
and are themselves float32 sums over K or N.
"""

from __future__ import annotations

import pytest
import torch

from opengenie_amd import _lib
from opengenie_amd import lora as A
from opengenie_amd import ltx_ops as L
from opengenie_amd.block import FP8Linear

from helpers import gen

F32 = 2.0 ** -24


def rnd(*shape, seed, dtype=torch.float32, device="cpu", std=1.0):
    return (torch.randn(shape, generator=gen(seed)) * std).to(dtype).to(device)


def case(rows, k, n, rank, adapters, dtype, device, seed=0):
    return {"x": rnd(rows, k, seed=seed, dtype=dtype, device=device), "y": rnd(rows, n, seed=seed + 1, dtype=dtype, device=device),
            "dy": rnd(rows, n, seed=seed + 2, dtype=dtype, device=device),
            "a": rnd(adapters, rank, k, seed=seed + 3, dtype=dtype, device=device, std=k ** -0.5),
            "b": rnd(adapters, n, rank, seed=seed + 4, dtype=dtype, device=device, std=0.2),
            "scale": rnd(adapters, seed=seed + 5, device=device)}


def segs(starts, ids, device, dtype=torch.int32):
    return torch.tensor(starts, dtype=dtype, device=device), torch.tensor(ids, dtype=dtype, device=device)


def exact(c, starts, ids):
    """Results in float64 and the bounds of the kernels' errors."""
    x, y, dy, a, b = (c[n].double() for n in ("x", "y", "dy", "a", "b"))
    scale = torch.ones(len(a), dtype=torch.float64, device=x.device) if c["scale"] is None else c["scale"].double()
    half = 2.0 ** -16 if c["x"].dtype == torch.bfloat16 else 2.0 ** -21
    tiny = 0.0 if c["x"].dtype == torch.bfloat16 else 2.0 ** -25
    k, n, rank = x.shape[1], y.shape[1], a.shape[1]
    r = {"y": y.clone(), "dx": torch.zeros_like(x), "da": torch.zeros_like(a), "db": torch.zeros_like(b)}
    e = {m: torch.zeros_like(t) for m, t in r.items()}
    count = {}
    for lo, hi, i in zip(starts, starts[1:], ids):
        if not 0 <= i < len(a) or hi <= lo:
            continue
        count[i] = count.get(i, 0) + hi - lo
        s, xs, dys = scale[i], x[lo:hi], dy[lo:hi]
        low, dlow = s * xs @ a[i].t(), s * dys @ b[i]
        elow = (k + 8) * F32 * s.abs() * xs.abs() @ a[i].abs().t() + half * low.abs() + tiny
        edlow = (n + 8) * F32 * s.abs() * dys.abs() @ b[i].abs() + half * dlow.abs() + tiny
        r["y"][lo:hi] += low @ b[i].t()
        e["y"][lo:hi] = (elow + (2 * rank + 2) * F32 * low.abs()) @ b[i].abs().t() + F32 * y[lo:hi].abs()
        r["dx"][lo:hi] = dlow @ a[i]
        e["dx"][lo:hi] = (edlow + (2 * rank + 2) * F32 * dlow.abs()) @ a[i].abs()
        r["da"][i] += dlow.t() @ xs
        e["da"][i] += (edlow + 2 * count[i] * F32 * dlow.abs()).t() @ xs.abs()
        r["db"][i] += dys.t() @ low
        e["db"][i] += dys.abs().t() @ (elow + 2 * count[i] * F32 * low.abs())
    u = torch.finfo(c["x"].dtype).eps / 2
    for m in r:
        e[m] = 1.01 * e[m] + u * (r[m].abs() + e[m]) + (tiny if tiny else 1e-37)
    return r, e


def run_and_check(c, starts, ids, dtype=torch.int32, out=None):
    st, sa = segs(starts, ids, c["x"].device, dtype)
    r, e = exact(c, starts, ids)
    y, low = A.lora_add(c["y"], c["x"], c["a"], c["b"], c["scale"], st, sa, save_low=True, out=out)
    got = (y, *A.lora_backward(c["dy"], c["x"], low, c["a"], c["b"], c["scale"], st, sa))
    for (name, want), t in zip(r.items(), got):
        assert t.dtype == c["x"].dtype and t.shape == want.shape
        off = ((t.double() - want).abs() - e[name]).max().item()
        assert off <= 0, f"{name}: {off:.3g} over the bound"
    return got


# ------------------------------------------------------------------- CPU
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("starts,ids", [([0, 5, 9], [1, 0]), ([2, 2, 7, 7], [0, 2, 1]), ([0, 9], [-1]),
                                        ([1, 3, 4, 8], [2, 7, 2])])
def test_torch_path_is_the_formulas(starts, ids, dtype):
    run_and_check(case(9, 12, 10, 3, 3, dtype, "cpu"), starts, ids, torch.int64)


def test_gradients_against_differences():
    c = {m: t.double() for m, t in case(7, 6, 5, 2, 3, torch.float64, "cpu").items()}
    st, sa = segs([0, 2, 6], [2, 0], "cpu")
    leaves = [c[m].requires_grad_(True) for m in ("y", "x", "a", "b")]
    scale = c["scale"].float()
    assert torch.autograd.gradcheck(lambda y, x, a, b: A.lora_add_with_grad(y, x, a, b, scale, st, sa), leaves)


def test_rows_without_an_adapter_keep_theirs():
    c = case(6, 8, 8, 2, 2, torch.bfloat16, "cpu")
    c["x"][4:] = float("nan")
    c["y"][5] = float("inf")
    c["dy"][4:] = float("nan")
    st, sa = segs([0, 2, 4, 5], [0, 1, -1], "cpu")
    y, low = A.lora_add(c["y"], c["x"], c["a"], c["b"], c["scale"], st, sa, save_low=True)
    assert torch.equal(y[4:], c["y"][4:])
    dx, da, db = A.lora_backward(c["dy"], c["x"], low, c["a"], c["b"], c["scale"], st, sa)
    assert not dx[4:].any() and torch.isfinite(da).all() and torch.isfinite(db).all()


def test_stacked_adapters_of_different_ranks():
    pairs = [(rnd(r, 16, seed=r), rnd(24, r, seed=r + 1), 0.5 * r) for r in (3, 8, 13)]
    ad = A.LoraAdapters.stack(pairs)
    assert ad.a.shape == (3, 16, 16) and ad.b.shape == (3, 24, 16) and ad.scale.tolist() == [1.5, 4.0, 6.5]
    x, y = rnd(9, 16, seed=1), rnd(9, 24, seed=2)
    st, sa = segs([0, 3, 6, 9], [0, 1, 2], "cpu")
    got = A.lora_add(y, x, ad.a, ad.b, ad.scale, st, sa)
    want = torch.cat([y[3 * i:3 * i + 3] + s * (x[3 * i:3 * i + 3] @ a.t()) @ b.t() for i, (a, b, s) in enumerate(pairs)])
    torch.testing.assert_close(got, want)


def test_empty_inputs():
    c = case(4, 8, 8, 2, 2, torch.bfloat16, "cpu")
    st, sa = segs([0], [], "cpu")
    y, low = A.lora_add(c["y"], c["x"], c["a"], c["b"], None, st, sa, save_low=True)
    assert torch.equal(y, c["y"]) and y.data_ptr() != c["y"].data_ptr() and low.shape == (4, 2)
    dx, da, db = A.lora_backward(c["dy"], c["x"], low, c["a"], c["b"], None, st, sa)
    assert not dx.any() and not da.any() and not db.any()
    st, sa = segs([0, 0], [1], "cpu")
    y, low = A.lora_add(c["y"][:0], c["x"][:0], c["a"], c["b"], None, st, sa, save_low=True)
    assert y.shape == (0, 8) and low.shape == (0, 2)
    dx, da, db = A.lora_backward(c["dy"][:0], c["x"][:0], low, c["a"], c["b"], None, st, sa)
    assert dx.shape == (0, 8) and not da.any() and not db.any()


def test_refusals():
    c = case(6, 8, 10, 2, 3, torch.bfloat16, "cpu")
    st, sa = segs([0, 2, 6], [0, 1], "cpu")
    ok = dict(y=c["y"], x=c["x"], a=c["a"], b=c["b"], scale=c["scale"], segment_starts=st, segment_adapters=sa)
    A.lora_add(**ok)
    for bad in ({"x": c["x"][:3]}, {"x": c["x"].float()}, {"y": c["y"].float()}, {"a": c["a"][0]}, {"a": c["a"][:2]},
                {"a": c["a"][:, :1]}, {"a": c["a"][:, :, :4]}, {"b": c["b"][:, :4]}, {"a": c["a"].half()},
                {"scale": c["scale"][:2]}, {"scale": c["scale"].double()}, {"segment_starts": st[:2]},
                {"segment_starts": st.float()}, {"segment_adapters": sa.bool()}, {"segment_adapters": sa[None]},
                {"out": c["y"][:3]}, {"out": c["y"].float()}, {"out": c["y"].t().contiguous().t()}):
        with pytest.raises(ValueError):
            A.lora_add(**{**ok, **bad})
    low = torch.zeros(6, 2)
    for dy, lw in ((c["dy"][:3], low), (c["dy"].float(), low), (c["dy"], low[:3]), (c["dy"], low.int())):
        with pytest.raises(ValueError):
            A.lora_backward(dy, c["x"], lw, c["a"], c["b"], c["scale"], st, sa)


@pytest.mark.skipif(not _lib.available(), reason="library not built")
def test_entry_points_refuse_what_the_kernels_do_not_take():
    """Nothing is launched: every call here fails its argument checks."""
    lib, p = _lib.load(), 4096

    def add(dt=0, y=p, ys=64, x=p, starts=p, ids=p, segments=1, adapters=1, low=p, rows=4, k=64, n=64, rank=8,
            ws=p, size=1 << 40):
        return lib.oga_lora_add(dt, y, ys, x, 64, p, p, None, starts, ids, segments, adapters, low, p, 64, rows, k, n,
                                rank, ws, size, None)

    for kw in ({"dt": 1}, {"y": None}, {"y": 4104}, {"ys": 60}, {"x": None}, {"starts": None}, {"ids": None},
               {"starts": 4098}, {"segments": 0}, {"adapters": 0}, {"adapters": 5000}, {"low": 4104}, {"rows": 0},
               {"k": 60}, {"n": 4}, {"k": 0}):
        assert add(**kw) == -1, kw
    for kw in ({"rank": 4}, {"rank": 12}, {"rank": 136}, {"rows": 1 << 31}, {"n": 1 << 23}):
        assert add(**kw) == -2, kw
    need = lib.oga_lora_add_workspace_bytes(4, 64, 8, 1)
    assert need > 0 and lib.oga_lora_add_workspace_bytes(4, 64, 136, 1) == 0
    assert add(ws=None) == -1 and add(ws=p + 16) == -1 and add(size=need - 1) == -1
    need = lib.oga_lora_bwd_workspace_bytes(4, 64, 64, 8, 1, 1)
    assert need > 0 and lib.oga_lora_bwd_workspace_bytes(4, 64, 64, 136, 1, 1) == 0

    def bwd(ws, size):
        return lib.oga_lora_bwd(0, p, 64, p, 64, p, p, p, None, p, p, 1, 1, p, 64, p, p, 4, 64, 64, 8, ws, size, None)

    assert bwd(None, need) == -1 and bwd(p, need - 1) == -1 and bwd(p + 16, need) == -1


@pytest.mark.skipif(not _lib.available(), reason="library not built")
def test_entry_points_refuse_grids_past_the_hardware_limit():
    """Nothing is launched: every call here fails its argument checks."""
    lib, p = _lib.load(), 4096
    for rows, n, segments in ((1 << 28, 64, 1), (1 << 20, 1 << 17, 1), (4, 1 << 16, 1 << 20)):
        assert lib.oga_lora_add(0, p, n, p, 64, p, p, None, p, p, segments, 1, p, p, n, rows, 64, n, 8, p, 1 << 60,
                                None) == -2
        assert lib.oga_lora_bwd(0, p, n, p, 64, p, p, p, None, p, p, segments, 1, p, 64, p, p, rows, 64, n, 8, p, 1 << 60,
                                None) == -2


@pytest.mark.skipif(not _lib.available(), reason="library not built")
def test_entry_points_refuse_row_strides_past_32_bit_offsets():
    """Nothing is launched: every call here fails its argument checks."""
    lib, p = _lib.load(), 4096
    for ys, outs in ((1 << 26, 64), (64, 1 << 26), (-64, 64), (64, -64)):
        assert lib.oga_lora_add(0, p, ys, p, 64, p, p, None, p, p, 1, 1, p, p, outs, 4, 64, 64, 8, p, 1 << 40, None) == -2
    for dys, xs, dxs in ((64, 64, 1 << 26), (64, 64, -64), (64, 1 << 26, 64), (1 << 26, 64, 64)):
        assert lib.oga_lora_bwd(0, p, dys, p, xs, p, p, p, None, p, p, 1, 1, p, dxs, p, p, 4, 64, 64, 8, p, 1 << 40,
                                None) == -2


# ------------------------------------------------------------------- GPU
SEGMENTS = [
    ([0, 1], [0]), ([0, 70], [1]), ([3, 3, 20, 64, 65, 67], [0, 1, 5, 2, -1]), ([0, 16, 32, 48, 64, 80], [2, 2, 0, 1, 2]),
    ([5, 60, 61, 129, 200], [1, 0, 0, 2]), (list(range(41)), [i % 4 - 1 for i in range(40)]),
    ([0, 300, 301, 640], [2, 0, 2]), (list(range(0, 281, 2)), [(7 * i) % 3 for i in range(140)]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 48, 64, 72, 128])
def test_gpu_against_float64(rank, dtype, monkeypatch):
    """Segments of every kind: empty ones, one row, ends inside and at a tile's
    end, rows before the first and behind the last, adapters that repeat, out
    of range and unused ones, more segments than a wave has lanes."""
    monkeypatch.setenv("OPENGENIE_AMD_STRICT", "1")
    L.reset_hip_calls()
    for i, (starts, ids) in enumerate(SEGMENTS):
        k, n = [(256, 512), (1032, 264), (8, 8), (520, 1048)][i % 4]
        c = case(starts[-1] + (i % 3) * 17, k, n, rank, 3, dtype, "cuda", seed=100 * i)
        if i % 2:
            c["scale"] = None
        run_and_check(c, starts, ids, torch.int64 if i % 3 == 0 else torch.int32)
    assert L.collect_hip_calls() == {"lora_add": len(SEGMENTS), "lora_backward": len(SEGMENTS)}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank", [8, 64, 128])
def test_gpu_long_segments_against_float64(rank, dtype):
    """Workgroups that stream several rounds of rows, whole and cut short, with
    and without an adapter, and columns that end inside a wave's 128."""
    for rows, k, n, starts, ids in ((6001, 72, 4104, [3, 2900, 5989], [1, 0]), (4999, 2056, 136, [0, 4000, 4500, 4999], [0, 7, 1])):
        c = case(rows, k, n, rank, 2, dtype, "cuda", seed=rows)
        want = run_and_check(c, starts, ids)
        y, rest = c["y"].clone(), (c["a"], c["b"], c["scale"], *segs(starts, ids, "cuda"))
        assert torch.equal(A.lora_add(y, c["x"], *rest, out=y), want[0])


@pytest.mark.gpu
def test_gpu_in_place_and_layouts_give_the_same_bits():
    c = case(150, 256, 320, 16, 2, torch.bfloat16, "cuda")
    st, sa = segs([0, 40, 130], [1, 0], "cuda")
    rest = (c["a"], c["b"], c["scale"], st, sa)
    want, low = A.lora_add(c["y"], c["x"], *rest, save_low=True)
    grads = A.lora_backward(c["dy"], c["x"], low, *rest)
    wide = torch.full((150, 600), float("nan"), device="cuda", dtype=torch.bfloat16)
    wide[:, 8:264] = c["x"]
    assert torch.equal(A.lora_add(c["y"], wide[:, 8:264], *rest), want)
    odd = torch.empty(c["y"].numel() + 1, device="cuda", dtype=torch.bfloat16)[1:].view(150, 320).copy_(c["y"])
    assert torch.equal(A.lora_add(odd, c["x"].view(3, 50, 256).flatten(0, 1), *rest), want)
    y3 = A.lora_add(c["y"].view(3, 50, 320), c["x"].view(3, 50, 256), *rest)
    assert torch.equal(y3.flatten(0, 1), want)
    dy = c["dy"].t().contiguous().t()
    for x, y in zip(A.lora_backward(dy, c["x"], low, *rest), grads):
        assert torch.equal(x, y)
    y = c["y"].clone()
    assert A.lora_add(y, c["x"], *rest, out=y) is y and torch.equal(y, want)


@pytest.mark.gpu
def test_gpu_padding_may_hold_anything():
    """Rows without an adapter hold infinities and NaN; they keep y, and no
    sum sees them."""
    c = case(200, 264, 320, 16, 3, torch.bfloat16, "cuda")
    starts, ids = [10, 60, 90, 170], [1, -1, 0]
    st, sa = segs(starts, ids, "cuda")
    rest = (c["a"], c["b"], c["scale"], st, sa)
    want, low = A.lora_add(c["y"], c["x"], *rest, save_low=True)
    grads = A.lora_backward(c["dy"], c["x"], low, *rest)
    out = torch.ones(200, dtype=torch.bool, device="cuda")
    out[10:60] = out[90:170] = False
    for t in (c["x"], c["y"], c["dy"]):
        t[out] = float("nan")
        t[out, ::3] = float("inf")
    got, low = A.lora_add(c["y"], c["x"], *rest, save_low=True)
    assert torch.equal(got[~out], want[~out])
    assert torch.equal(got[out].view(torch.int16), c["y"][out].view(torch.int16))
    for x, y in zip(A.lora_backward(c["dy"], c["x"], low, *rest), grads):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_gpu_starts_that_do_not_rise_stay_within_the_tensors():
    """Rows of requests with sound starts keep their results, whatever the
    others hold; the rest is undefined and inside the outputs."""
    c = case(96, 64, 64, 8, 2, torch.bfloat16, "cuda")
    guard = torch.full((3, 96, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    for starts, ids in (([50, 20, 96], [0, 1]), ([-40, 30, 5000], [1, 0]), ([96, 0], [1]),
                        ([2 ** 31 - 1, -2 ** 31], [0]), ([0, 96], [2 ** 31 - 1]), ([0, 96], [-2 ** 31])):
        st, sa = segs(starts, ids, "cuda")
        out, low = A.lora_add(c["y"], c["x"], c["a"], c["b"], c["scale"], st, sa, out=guard[1], save_low=True)
        A.lora_backward(c["dy"], c["x"], low, c["a"], c["b"], c["scale"], st, sa)
        torch.cuda.synchronize()
        assert (guard[0] == 7).all() and (guard[2] == 7).all()
    assert torch.equal(guard[1], c["y"])  # the last one has no adapter


@pytest.mark.gpu
def test_gpu_same_bits_twice_in_a_graph_and_on_another_stream():
    c = case(333, 512, 256, 32, 3, torch.bfloat16, "cuda")
    other = case(333, 512, 256, 32, 3, torch.bfloat16, "cuda", seed=50)
    st, sa = segs([0, 100, 333], [2, 0], "cuda")
    st2, sa2 = segs([7, 200, 300], [1, 1], "cuda")

    def step(c, st, sa):
        y, low = A.lora_add(c["y"], c["x"], c["a"], c["b"], c["scale"], st, sa, save_low=True)
        return (y, *A.lora_backward(c["dy"], c["x"], low, c["a"], c["b"], c["scale"], st, sa))

    want, want2 = step(c, st, sa), step(other, st2, sa2)
    static, sst, ssa = {m: t.clone() for m, t in c.items()}, st.clone(), sa.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for x, y in zip(want, step(static, sst, ssa)):
            assert torch.equal(x, y)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(static, sst, ssa)
    for fresh, fst, fsa, expect in ((other, st2, sa2, want2), (c, st, sa, want)) * 2:
        for m, t in fresh.items():
            static[m].copy_(t)
        sst.copy_(fst)
        ssa.copy_(fsa)
        graph.replay()
        torch.cuda.synchronize()
        step(c, st2, sa)
        for x, y in zip(got, expect):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_gpu_fp8_linear_with_adapters():
    w, x = rnd(512, 256, seed=1, device="cuda", std=0.05), rnd(2, 30, 256, seed=2, dtype=torch.bfloat16, device="cuda")
    lin = FP8Linear.quantized(w, 8.0 / 448, rnd(512, seed=3, dtype=torch.bfloat16, device="cuda"))
    c = case(60, 256, 512, 16, 2, torch.bfloat16, "cuda")
    st, sa = segs([0, 30, 60], [1, 0], "cuda")
    got = A.fp8_linear_lora_forward(lin, x, A.LoraAdapters(c["a"], c["b"], c["scale"]), st, sa)
    want = A.lora_add(L.fp8_linear_forward(lin, x), x, c["a"], c["b"], c["scale"], st, sa)
    assert got.shape == (2, 30, 512) and torch.equal(got, want)
