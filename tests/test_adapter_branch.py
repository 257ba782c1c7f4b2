"""The operators of a fine-tuned attention branch run together: FP8
projections with adapters beside them, head norms and rotation, attention with
gradients, back to the adapters and the norm weights."""

from __future__ import annotations

import pytest
import torch

from opengenie_amd import attention_grad as G
from opengenie_amd import head_rope as H
from opengenie_amd import lora as A
from opengenie_amd import ltx_ops as L
from opengenie_amd.block import FP8Linear
from opengenie_amd.rope import rotary_cos_sin

from helpers import gen

B, N, DIM, HEADS, KV, HD, RANK, REQ = 2, 75, 256, 4, 2, 64, 16, 3


def rnd(*shape, seed, dtype=torch.float32, std=1.0, mean=0.0):
    return torch.randn(shape, generator=gen(seed)).mul(std).add(mean).to(dtype)


def make(device):
    p = {"x": rnd(B, N, DIM, seed=1, dtype=torch.bfloat16), "dout": rnd(B, N, HEADS, HD, seed=2, dtype=torch.bfloat16)}
    for i, (name, out) in enumerate((("q", HEADS * HD), ("k", KV * HD), ("v", KV * HD))):
        p["w" + name] = rnd(out, DIM, seed=10 + i, std=DIM ** -0.5)
        p["a" + name] = rnd(REQ, RANK, DIM, seed=20 + i, std=DIM ** -0.5, dtype=torch.bfloat16)
        p["b" + name] = rnd(REQ, out, RANK, seed=30 + i, std=0.2, dtype=torch.bfloat16)
    p["qn"], p["kn"] = rnd(HD, seed=40, std=0.1, mean=1.0), rnd(HD, seed=41, std=0.1, mean=1.0)
    p = {n: t.to(device) for n, t in p.items()}
    p["scale"] = torch.tensor([1.0, 0.5, 2.0], device=device)
    p["starts"] = torch.tensor([0, 60, 90, 2 * N - 5], device=device, dtype=torch.int32)
    p["ids"] = torch.tensor([2, 0, 1], device=device, dtype=torch.int32)
    p["lens"] = torch.tensor([N, N - 20], device=device, dtype=torch.int32)
    p["cos"], p["sin"] = rotary_cos_sin(N, 32, device=device)
    return p


def branch(p, base, wide=None):
    """The branch's output and gradients. `base` gives the frozen projections;
    with `wide`, every tensor in that dtype."""
    def c(t):
        return t if wide is None or not t.is_floating_point() else t.to(wide)

    leaves = {n: c(p[n]).detach().requires_grad_(True) for n in ("x", "aq", "bq", "ak", "bk", "av", "bv", "qn", "kn")}
    heads = {}
    for name, h in (("q", HEADS), ("k", KV), ("v", KV)):
        y = A.lora_add_with_grad(c(base[name]), leaves["x"], leaves["a" + name], leaves["b" + name], p["scale"],
                                 p["starts"], p["ids"])
        heads[name] = y.view(B, N, h, HD)
    q, k = H.qk_head_rmsnorm_rope_with_grad(heads["q"], heads["k"], leaves["qn"], leaves["kn"], 1e-6, c(p["cos"]),
                                            c(p["sin"]), layout="interleaved")
    out = G.attention_with_grad(q, k, heads["v"], None, True, p["lens"])
    out.backward(c(p["dout"]))
    return {"out": out.detach(), **{n: t.grad for n, t in leaves.items()}}


@pytest.mark.gpu
def test_branch_against_float64(monkeypatch):
    """Every result against the same branch in float64. Between the inputs and
    a gradient lie at most eight roundings to bf16 (projection with adapter,
    norm, P or out, out in Delta, dS, dq, the norm's gradient, the result): in
    2-norms each adds at most 2^-8 of the norm of what it rounds, and norms and
    rotations keep their sizes, so 8 x 2^-8 of the result's norm."""
    monkeypatch.setenv("OPENGENIE_AMD_STRICT", "1")
    p = make("cuda")
    lin = {n: FP8Linear.quantized(p["w" + n], 8.0 / 448, None) for n in "qkv"}
    base = {n: L.fp8_linear_forward(lin[n], p["x"]) for n in "qkv"}
    got = branch(p, base)
    monkeypatch.delenv("OPENGENIE_AMD_STRICT")
    want = branch({n: t.cpu() for n, t in p.items()}, {n: t.cpu() for n, t in base.items()}, torch.float64)
    for n, t in got.items():
        w = want[n]
        off = (t.double().cpu() - w).norm() / w.norm()
        assert off <= 8 * 2.0 ** -8, f"{n}: {off:.3g}"
        assert w.norm() > 0


def test_branch_on_the_cpu_in_both_precisions():
    """The branch of torch paths: float32 leaves against float64 ones (float32
    roundings, at most 2^-16 of a result's norm here)."""
    p = make("cpu")
    base = {n: p["x"].float() @ p["w" + n].t() for n in "qkv"}
    got, want = branch(p, base, torch.float32), branch(p, base, torch.float64)
    for n, w in want.items():
        assert (got[n].double() - w).norm() <= 2.0 ** -16 * w.norm(), n


@pytest.mark.gpu
def test_branch_serves_single_tokens():
    """One new token of each request: adapters, norms at each request's
    position, and attention over its own padded keys, in one captured graph,
    against eager calls."""
    reqs, keys = 5, 40
    x = rnd(reqs, 1, DIM, seed=50, dtype=torch.bfloat16).cuda()
    lin = FP8Linear.quantized(rnd(HEADS * HD, DIM, seed=51, std=DIM ** -0.5).cuda(), 8.0 / 448, None)
    ad = A.LoraAdapters(rnd(3, 8, DIM, seed=52, std=DIM ** -0.5, dtype=torch.bfloat16).cuda(),
                        rnd(3, HEADS * HD, 8, seed=53, dtype=torch.bfloat16).cuda())
    starts = torch.arange(reqs + 1, device="cuda", dtype=torch.int32)
    ids = torch.tensor([0, 2, -1, 1, 2], device="cuda", dtype=torch.int32)
    k, v = (rnd(reqs, keys, KV, HD, seed=54 + i, dtype=torch.bfloat16).cuda() for i in range(2))
    lens = torch.tensor([1, 40, 17, 33, 2], device="cuda", dtype=torch.int32)
    pos = (lens - 1).view(reqs, 1)
    w = rnd(HD, seed=56, mean=1.0, std=0.1).cuda()
    cos, sin = rotary_cos_sin(keys, HD, device="cuda")

    def step():
        q = A.fp8_linear_lora_forward(lin, x, ad, starts, ids).view(reqs, 1, HEADS, HD)
        q, kk = H.qk_head_rmsnorm_rope(q, k[:, :1], w, w, 1e-6, cos, sin, positions=pos)
        return q, kk, G.flash_attn_lse(q, k, v, causal=True, k_lens=lens)[0]

    want = [t.clone() for t in step()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    keep = x.clone()
    for i in range(4):
        x.copy_(keep if i % 2 else keep * 2)
        expect = want if i % 2 else [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, expect):
            assert torch.equal(a, b)
