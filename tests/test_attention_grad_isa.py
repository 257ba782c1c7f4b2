"""Properties of the compiled code of the attention gradients that GPU runs
cannot pin down reliably (CPU only: hipcc cross-compiles, nothing is launched).

The three kernels bring tiles into LDS by DMA, which vmcnt counts, and read
them with inline-assembly ds_read instructions after a barrier: each barrier
needs a wait for the tile that the step reads, and no instruction may name a
register that a read in flight will still write. What the wait may leave in
flight is what one step sends after the tile it reads: a tile pair is
2 x 64 rows of 2 D bytes, in pieces of 1024 bytes a wave, and k_attn_dkv sends
a piece of (lse, Delta) beside it.
"""

from __future__ import annotations

import os
import re

import pytest

from test_kernel_isa import CSRC, _device_asm, _kernel_body, barrier_violations, lds_read_hazards

hipcc_needed = pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc") and not os.environ.get("HIPCC"),
                                  reason="hipcc not present")
FORMS = [(k, d, w, bufs, causal)
         for k in ("k_attn_lse", "k_attn_dq", "k_attn_dkv")
         for d, w, bufs in ((64, 4, 3), (128, 8, 3), (128, 4, 2))
         for causal in (0, 1)]


def _body(k, d, w, bufs, causal):
    asm = _device_asm(os.path.join(CSRC, "attention_grad.hip"))
    return _kernel_body(asm, f"{k}ILi{d}ELi{w}ELi{bufs}ELb{causal}E")


@hipcc_needed
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_barriers_wait_for_the_tiles_dma(form):
    k, d, w, bufs, _ = form
    body = _body(*form)
    step = 2 * (64 * 2 * d // 1024) // w + (k == "k_attn_dkv")
    assert sum(1 for ins in body if ins == "s_barrier") >= 1
    assert sum("load_lds" in ins for ins in body) >= step
    assert barrier_violations(body, max_vmcnt=step if bufs == 3 else 0) == []


@hipcc_needed
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_no_register_of_an_outstanding_lds_read_is_named(form):
    assert lds_read_hazards(_body(*form)) == []


@hipcc_needed
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_main_loop_holds_its_registers(form):
    """No scratch access between the label and the branch of the smallest loop
    with matrix instructions and a barrier, the walk over the tiles."""
    body = _body(*form)
    labels = {ins[:-1]: i for i, ins in enumerate(body) if ins.endswith(":")}
    back = [(labels[m.group(1)], i) for i, ins in enumerate(body)
            if (m := re.match(r"s_c?branch\w*\s+(\S+)", ins)) and labels.get(m.group(1), i) < i]
    loops = [body[a:b] for a, b in back
             if "s_barrier" in body[a:b] and sum("mfma" in ins for ins in body[a:b]) >= 16]
    loop = min(loops, key=len)
    assert not [ins for ins in loop if ins.startswith("scratch_")]
