"""Gradients of attention rows that see few keys, in float64.

There out is as large as the values, and Delta summed from the rounded out is
off by up to 2^-8 sum |dout| |out|, far more than dP - Delta where the values
of the keys are alike. The kernel corrects Delta by the row's sum of
P (dP - Delta), so that only float32 errors are left in it: of dP - Delta, a
sum of D products and Delta, (D + 3) 2^-24 of the terms' absolute sum; of the
correction, the same and P's relative error `rel` (twice: numerator and
denominator) of the largest difference. dS is then rounded once to bf16 (u =
2^-8), and the results once. (Rows of up to 48 keys, and a causal sequence's rows
up to the 128th key, are corrected.)
"""

from __future__ import annotations

import pytest
import torch

from opengenie_amd import attention_grad as G

from helpers import gen
from test_attention_grad import F32, U

pytestmark = pytest.mark.gpu


def alike(b, nq, nk, h, hk, d, seed):
    """Values that differ by an eighth of their size from key to key."""
    g = gen(seed)
    q, do = (torch.randn((b, nq, h, d), generator=g) for _ in range(2))
    k = torch.randn((b, nk, hk, d), generator=g)
    v = torch.randn((b, 1, hk, d), generator=g) + torch.randn((b, nk, hk, d), generator=g) / 8
    return [t.bfloat16().cuda() for t in (q, k, v, do)]


FEW = [(2, 3, 1, 2, 2, 128), (1, 70, 2, 4, 2, 64), (2, 33, 5, 2, 1, 128), (1, 1, 9, 4, 2, 64), (1, 300, 33, 2, 2, 128),
       (1, 150, 48, 2, 1, 64)]
CAUSAL = [(1, 300, 64, 2, 2, 128), (2, 90, 90, 2, 1, 64), (1, 127, 100, 2, 2, 128), (1, 128, 128, 1, 1, 64),
          (1, 20, 125, 2, 2, 128)]


@pytest.mark.parametrize("shape,causal", [(s, c) for s in FEW for c in (False, True)] + [(s, True) for s in CAUSAL])
def test_small_differences_are_kept(shape, causal):
    b, nq, nk, h, hk, d = shape
    q, k, v, do = alike(*shape, seed=nq + nk)
    scale = d ** -0.5
    out, lse = G.flash_attn_lse(q, k, v, causal=causal)
    dq, dk, _ = G.flash_attn_backward(do, q, k, v, out, lse, causal=causal)
    want_k, off_k = (torch.zeros(k.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for i in range(b):
        for j in range(h):
            c = j // (h // hk)
            x, kk, vv, g = (t.double() for t in (q[i, :, j], k[i, :, c], v[i, :, c], do[i, :, j]))
            s = x @ kk.t() * scale
            if causal:
                s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(nk - nq + 1), float("-inf"))
            some = (s > float("-inf")).any(1)
            x, g, s = x[some], g[some], s[some]
            assert not dq[i, ~some, j].any()
            p = torch.softmax(s, 1)
            seen = p > 0
            o, dp = p @ vv, g @ vv.t()
            delta = (g * o).sum(1, keepdim=True)
            diff = torch.where(seen, dp - delta, 0.0)
            size = g.abs() @ vv.abs().t()
            rel = 2 * ((d + 2) * F32 * scale * (x.abs() @ kk.abs().t()) * seen).amax(1, keepdim=True) + 2.0 ** -20
            eg = (d + 3) * F32 * (size + delta.abs()) * seen
            rough = U * (g.abs() * o.abs()).sum(1, keepdim=True) * 1.01  # of Delta before it is corrected
            er = eg.amax(1, keepdim=True) + 2 * rel * (diff.abs().amax(1, keepdim=True) + rough)
            ds = p * diff
            eds = ((U + rel) * ds.abs() + p * (eg + er) * (1 + U)) * 1.01
            want, off = scale * (ds @ kk), scale * (eds @ kk.abs()) * 1.01
            assert ((dq[i, some, j].double() - want).abs() <= off + U * (want.abs() + off) + 1e-30).all()
            want_k[i, :, c] += scale * (ds.t() @ x)
            off_k[i, :, c] += scale * (eds.t() @ x.abs()) * 1.01
    assert ((dk.double() - want_k).abs() <= off_k + U * (want_k.abs() + off_k) + 1e-30).all()
