"""Timed operators of an attention branch that is fine-tuned and served with
adapters, on one GPU: attention with its gradients, the norms of queries and
keys for each head with the position rotation (and the rotation alone), and
low-rank adapters of many requests beside a shared projection.

listed() names the cases, draw(rng) gives one more of the same ranges,
prepare() makes what the program holds before the call, run() makes the call:
in its plain form (elementary torch operations in float32, 64 bits for long
sums, rounded once) or, with `own`, through `opengenie_amd`. work() counts
what the call cannot do without and exact() evaluates it in float64.

Sizes are those of the video block (hidden size 4096, 32 heads of 128,
feed-forward width 16384, 9216 tokens of a 576p clip, 2304 of a quarter-size
one, prompts of 256 tokens) and of its audio branch (hidden size 2048, 32
heads of 64), or generic."""

import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------
def listed():
    return [
        # Attention, forward and backward.
        # One query per sequence (a pooled or newest token) on four padded
        # sequences: the smallest call of a step, where latency counts.
        {"name": "attn_step_4x1x577", "op": "attention", "batch": 4, "nq": 1, "nk": 577, "heads": 32, "kv_heads": 8,
         "dim": 128, "causal": True, "padded": True},
        # Text cross-attention of two quarter-size clips whose prompts have
        # different lengths in one padded batch.
        {"name": "attn_text_2x2304x256", "op": "attention", "batch": 2, "nq": 2304, "nk": 256, "heads": 32,
         "kv_heads": 32, "dim": 128, "causal": False, "padded": True},
        # Causal attention with shared key/value heads of 64 at a length that
        # divides nothing.
        {"name": "attn_causal_4099", "op": "attention", "batch": 1, "nq": 4099, "nk": 4099, "heads": 32, "kv_heads": 8,
         "dim": 64, "causal": True, "padded": False},
        # Self-attention of the 576p clip.
        {"name": "attn_self_9216", "op": "attention", "batch": 1, "nq": 9216, "nk": 9216, "heads": 32, "kv_heads": 32,
         "dim": 128, "causal": False, "padded": False},
        # Head norms and rotation.
        # One new token of each of 32 requests, each at a position of its own.
        {"name": "rope_step_32x1", "op": "norm_rope", "batch": 32, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "layout": "half", "positions": True, "table": "f32", "weight": "bf16", "dtype": "bf16",
         "train": False},
        # The rotation alone, pairs of neighbours, over half of each head:
        # the keys of two long contexts.
        {"name": "rotate_2x8209", "op": "rotate", "batch": 2, "tokens": 8209, "heads": 8, "dim": 128, "rotary": 64,
         "layout": "interleaved", "positions": True, "table": "f32", "dtype": "bf16"},
        # Forward pass over a 576p clip.
        {"name": "norm_rope_9216", "op": "norm_rope", "batch": 1, "tokens": 9216, "heads": 32, "kv_heads": 32,
         "dim": 128, "rotary": 128, "layout": "half", "positions": False, "table": "f32", "weight": "bf16",
         "dtype": "bf16", "train": False},
        # A training step's forward and backward at an odd length, heads of
        # 64, three quarters of each rotated.
        {"name": "norm_rope_train_4999", "op": "norm_rope", "batch": 1, "tokens": 4999, "heads": 32, "kv_heads": 32,
         "dim": 64, "rotary": 48, "layout": "half", "positions": False, "table": "f32", "weight": "f32",
         "dtype": "bf16", "train": True},
        # Adapters.
        # One token of each of 32 requests over 16 adapters.
        {"name": "lora_step_32x1", "op": "lora", "tokens": 32, "requests": 32, "adapters": 16, "rank": 16, "k": 4096,
         "n": 4096, "dtype": "bf16", "train": False},
        # Ragged requests through the feed-forward up-projection.
        {"name": "lora_ragged_2305", "op": "lora", "tokens": 2305, "requests": 9, "adapters": 6, "rank": 32, "k": 4096,
         "n": 16384, "dtype": "bf16", "train": False},
        # Two 576p clips' halves with an adapter each.
        {"name": "lora_9216", "op": "lora", "tokens": 9216, "requests": 2, "adapters": 2, "rank": 64, "k": 4096,
         "n": 4096, "dtype": "bf16", "train": False},
        # A training step of three adapters on ragged sequences.
        {"name": "lora_train_4608", "op": "lora", "tokens": 4608, "requests": 5, "adapters": 3, "rank": 32, "k": 4096,
         "n": 4096, "dtype": "bf16", "train": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "norm_rope", "norm_rope", "rotate", "lora", "lora", "lora"])
    if op == "attention":
        # queries from one to a clip, keys of a prompt or of the same length
        heads, kv_heads = rng.choice([(32, 32), (32, 32), (32, 8), (16, 2), (8, 8)])
        nq = _log_int(rng, 1, 5000)
        nk = rng.choice([nq, _log_int(rng, 1, 1024), _log_int(rng, 64, 5000)])
        return {"op": op, "batch": rng.choice([1, 1, 2, 3]), "nq": nq, "nk": nk, "heads": heads, "kv_heads": kv_heads,
                "dim": rng.choice([64, 128, 128]), "causal": rng.random() < 0.4, "padded": rng.random() < 0.4}
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "norm_rope":
        dim = rng.choice([64, 128, 128, 256])
        heads, kv_heads = rng.choice([(32, 32), (32, 8), (16, 2), (24, 8)])
        return {"op": op, "batch": rng.choice([1, 1, 2, 5]), "tokens": _log_int(rng, 1, 4000), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "rotary": rng.randint(1, dim // 16) * 16,
                "layout": rng.choice(["half", "interleaved"]), "positions": rng.random() < 0.5,
                "table": rng.choice(["f32", "f32", "bf16"]), "weight": rng.choice(["bf16", "f32", "none"])
                if dtype == "bf16" else rng.choice(["f32", "none"]), "dtype": dtype, "train": rng.random() < 0.6}
    if op == "rotate":
        dim = rng.choice([64, 128, 128, 256])
        return {"op": op, "batch": rng.choice([1, 2, 3]), "tokens": _log_int(rng, 1, 8000), "heads": rng.choice([1, 8, 24]),
                "dim": dim, "rotary": rng.randint(1, dim // 16) * 16, "layout": rng.choice(["half", "interleaved"]),
                "positions": rng.random() < 0.5, "table": rng.choice(["f32", "bf16"]), "dtype": dtype}
    tokens = _log_int(rng, 1, 6000)
    k, n = rng.choice([(4096, 4096), (4096, 16384), (16384, 4096), (2048, 4096), (2056, 1032)])
    return {"op": op, "tokens": tokens, "requests": rng.randint(1, min(tokens, 40)), "adapters": rng.randint(1, 20),
            "rank": rng.choice([8, 16, 24, 32, 64, 128]), "k": k, "n": n, "dtype": dtype, "train": rng.random() < 0.5}


def _key_lengths(case):
    """Valid keys of each sequence: a padded batch's last sequence is whole."""
    b, nk = case["batch"], case["nk"]
    return [max(1, nk * (2 * i + 3) // (2 * b + 1)) for i in range(b)] if case["padded"] else [nk] * b


def _segments(case):
    """Row ranges of the requests: ragged, with a few rows of padding behind
    the last one where there are rows to spare."""
    t, s = case["tokens"], case["requests"]
    if t == s:
        return list(range(t + 1))
    rng = random.Random(t * 1009 + s)
    used = t - min(t // 50, t - s)
    return [0] + sorted(rng.sample(range(1, used), s - 1)) + [used]


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed))

    def normal(self, *shape, std=1.0, mean=0.0, dtype=torch.bfloat16):
        t = torch.randn(shape, generator=self.g, device=DEV, dtype=torch.float32)
        return t.mul_(std).add_(mean).to(dtype)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device=DEV, dtype=torch.int32)


def prepare(case, seed):
    r, op = _Rand(seed), case["op"]
    s = {"op": op, "case": dict(case)}
    if op == "attention":
        b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        s["q"], s["dout"] = r.normal(b, case["nq"], h, d), r.normal(b, case["nq"], h, d)
        s["k"], s["v"] = r.normal(b, case["nk"], hk, d), r.normal(b, case["nk"], hk, d)
        s["k_lens"] = torch.tensor(_key_lengths(case), device=DEV, dtype=torch.int32) if case["padded"] else None
        return s
    dt = DTYPES[case["dtype"]]
    if op == "lora":
        t, n, k, rank, ad = case["tokens"], case["n"], case["k"], case["rank"], case["adapters"]
        s["x"], s["y"] = r.normal(t, k, dtype=dt), r.normal(t, n, dtype=dt)
        s["a"] = r.normal(ad, rank, k, std=k ** -0.5, dtype=dt)
        s["b"] = r.normal(ad, n, rank, std=0.05, dtype=dt)
        s["scale"] = r.normal(ad, std=0.25, mean=1.0, dtype=torch.float32)
        s["starts"] = torch.tensor(_segments(case), device=DEV, dtype=torch.int32)
        s["ids"] = r.ints(0, ad, case["requests"])
        if case["train"]:
            s["dy"] = r.normal(t, n, dtype=dt)
        return s
    b, n, d, rot = case["batch"], case["tokens"], case["dim"], case["rotary"]
    length = 4 * n + 1000 if case["positions"] else n
    freq = 10000.0 ** (-torch.arange(rot // 2, device=DEV, dtype=torch.float64) * 2 / rot)
    angle = torch.arange(length, device=DEV, dtype=torch.float64)[:, None] * freq
    s["cos"], s["sin"] = angle.cos().to(DTYPES[case["table"]]), angle.sin().to(DTYPES[case["table"]])
    s["positions"] = None
    if case["positions"]:  # consecutive tokens from a start of each sequence's own
        s["positions"] = r.ints(0, length - n, b, 1) + torch.arange(n, device=DEV, dtype=torch.int32)
    if op == "rotate":
        s["x"] = r.normal(b, n, case["heads"], d, dtype=dt)
        return s
    s["q"], s["k"] = r.normal(b, n, case["heads"], d, dtype=dt), r.normal(b, n, case["kv_heads"], d, dtype=dt)
    s["qw"] = s["kw"] = None
    if case["weight"] != "none":
        wdt = DTYPES[case["weight"]]
        s["qw"], s["kw"] = r.normal(d, std=0.1, mean=1.0, dtype=wdt), r.normal(d, std=0.1, mean=1.0, dtype=wdt)
    if case["train"]:
        s["dq"], s["dk"] = r.normal(b, n, case["heads"], d, dtype=dt), r.normal(b, n, case["kv_heads"], d, dtype=dt)
    return s


# --------------------------------------------------------------------------
# the call
# --------------------------------------------------------------------------
def run(s):
    return {"attention": _attention, "norm_rope": _norm_rope, "rotate": _rotate, "lora": _lora}[s["op"]](s)


def _attention(s):
    c = s["case"]
    if own:
        from opengenie_amd import attention_grad as G

        out, lse = G.flash_attn_lse(s["q"], s["k"], s["v"], causal=c["causal"], k_lens=s["k_lens"])
        dq, dk, dv = G.flash_attn_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, causal=c["causal"],
                                           k_lens=s["k_lens"])
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    group, scale = c["heads"] // c["kv_heads"], c["dim"] ** -0.5
    q, do = (s[n].float().transpose(1, 2).contiguous() for n in ("q", "dout"))
    k, v = (s[n].float().transpose(1, 2).repeat_interleave(group, 1) for n in ("k", "v"))
    hide = _hidden(c, s["k_lens"])
    x = torch.matmul(q, k.transpose(2, 3)).mul_(scale)
    if hide is not None:
        x = x.masked_fill_(hide, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (m + total.log()).squeeze(-1)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    out = torch.matmul(p, v)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3))
    ds = ds.sub_((do * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3), q)
    dk, dv = (t.unflatten(1, (c["kv_heads"], group)).sum(2) for t in (dk, dv))
    out, dq, dk, dv = (t.transpose(1, 2).contiguous().to(s["q"].dtype) for t in (out, dq, dk, dv))
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _hidden(c, k_lens):
    """Keys each query does not see ([B, 1, Nq, Nk]): behind the sequence's
    length and, causal, later than the query, whose sequence ends with the
    last valid key."""
    if k_lens is None and not c["causal"]:
        return None
    j = torch.arange(c["nk"], device=DEV)
    lens = k_lens if k_lens is not None else torch.full((c["batch"],), c["nk"], device=DEV)
    lens = lens.long().view(-1, 1, 1, 1)
    hide = j >= lens
    if c["causal"]:
        hide = hide | (j > torch.arange(c["nq"], device=DEV)[:, None] + lens - c["nq"])
    return hide


def _tables(s, dtype):
    """cos and sin of each token, [B or 1, N, 1, R / 2]."""
    if s["positions"] is None:
        return tuple(s[n].to(dtype)[None, :, None, :] for n in ("cos", "sin"))
    return tuple(s[n].to(dtype)[s["positions"].long()][:, :, None, :] for n in ("cos", "sin"))


def _turn(x, cos, sin, layout):
    rot = 2 * cos.shape[-1]
    head, rest = x[..., :rot], x[..., rot:]
    if layout == "half":
        a, b = head[..., : rot // 2], head[..., rot // 2:]
        head = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((head, rest), -1)


def _rotate(s):
    if own:
        from opengenie_amd import head_rope as H

        return H.apply_rope(s["x"], s["cos"], s["sin"], layout=s["case"]["layout"], positions=s["positions"])
    cos, sin = _tables(s, torch.float32)
    return _turn(s["x"].float(), cos, sin, s["case"]["layout"]).to(s["x"].dtype)


def _norm_rope(s):
    c = s["case"]
    if own:
        from opengenie_amd import head_rope as H

        q, k = H.qk_head_rmsnorm_rope(s["q"], s["k"], s["qw"], s["kw"], EPS, s["cos"], s["sin"], layout=c["layout"],
                                      positions=s["positions"])
        if not c["train"]:
            return {"q": q, "k": k}
        dq, dk, dqw, dkw = H.qk_head_rmsnorm_rope_backward(
            s["dq"], s["dk"], s["q"], s["k"], s["qw"], s["kw"], EPS, s["cos"], s["sin"], layout=c["layout"],
            positions=s["positions"])
        return {"q": q, "k": k, "dq": dq, "dk": dk, "dqw": dqw, "dkw": dkw}
    cos, sin = _tables(s, torch.float32)
    r = {}
    x, w = s["q"].float(), s["qw"]
    r["q"], inv = _norm_turn(x, w, cos, sin, c["layout"])
    if c["train"]:
        r["dq"], r["dqw"] = _norm_turn_grad(s["dq"].float(), x, inv, w, cos, sin, c["layout"])
    x, w = s["k"].float(), s["kw"]
    r["k"], inv = _norm_turn(x, w, cos, sin, c["layout"])
    if c["train"]:
        r["dk"], r["dkw"] = _norm_turn_grad(s["dk"].float(), x, inv, w, cos, sin, c["layout"])
    dt = s["q"].dtype
    return {n: t.to(dt) if n in ("q", "k", "dq", "dk") else t for n, t in r.items()}


def _norm_turn(x, w, cos, sin, layout):
    inv = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    y = x * inv if w is None else x * inv * w.float()
    return _turn(y, cos, sin, layout), inv


def _norm_turn_grad(dy, x, inv, w, cos, sin, layout):
    dy = _turn(dy, cos, -sin, layout)
    n = x * inv
    dw = None if w is None else (dy * n).sum((0, 1, 2), dtype=torch.float64).to(w.dtype)
    g = dy if w is None else dy * w.float()
    return inv * (g - n * (g * n).mean(-1, keepdim=True)), dw


def _lora(s):
    c = s["case"]
    if own:
        from opengenie_amd import lora as A

        if not c["train"]:
            return A.lora_add(s["y"], s["x"], s["a"], s["b"], s["scale"], s["starts"], s["ids"])
        y, low = A.lora_add(s["y"], s["x"], s["a"], s["b"], s["scale"], s["starts"], s["ids"], save_low=True)
        dx, da, db = A.lora_backward(s["dy"], s["x"], low, s["a"], s["b"], s["scale"], s["starts"], s["ids"])
        return {"y": y, "dx": dx, "da": da, "db": db}
    # the products with every adapter, of which a row keeps its own
    ad, rank, dt = c["adapters"], c["rank"], s["x"].dtype
    row = torch.arange(c["tokens"], device=DEV, dtype=torch.int32)
    seg = torch.searchsorted(s["starts"], row, right=True) - 1
    mine = s["ids"][seg.clamp(max=c["requests"] - 1)].long()
    keep = torch.nn.functional.one_hot(mine, ad).float() * (row < s["starts"][-1])[:, None] * s["scale"]
    keep = keep.repeat_interleave(rank, 1)  # [T, adapters * rank]
    x, a = s["x"].float(), s["a"].float().flatten(0, 1)
    b = s["b"].float().transpose(1, 2).flatten(0, 1)  # [adapters * rank, N]
    low = torch.matmul(x, a.t()) * keep
    y = (s["y"].float() + torch.matmul(low, b)).to(dt)
    if not c["train"]:
        return y
    dy = s["dy"].float()
    dlow = torch.matmul(dy, b.t()) * keep
    dx, da = torch.matmul(dlow, a), torch.matmul(dlow.t(), x)
    db = torch.matmul(low.t(), dy).unflatten(0, (ad, rank)).transpose(1, 2).contiguous()
    return {"y": y, "dx": dx.to(dt), "da": da.unflatten(0, (ad, rank)).to(dt), "db": db.to(dt)}


# --------------------------------------------------------------------------
# the work, and the values in 64 bits
# --------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "attention":
        b, h, hk, d, nq, nk = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "nq", "nk"))
        pairs = 0
        for n in _key_lengths(case):
            if not case["causal"]:
                pairs += nq * n
            else:  # query i sees i + 1 + n - nq keys where that is positive
                first = max(0, nq - n)
                rows = nq - first
                pairs += rows * (first + 1 + n - nq + n) // 2
        # q, dout read, out, dq written; k, v read (the valid ones), dk, dv written; lse written
        valid = sum(_key_lengths(case))
        moved = 2 * (4 * b * nq * h * d + 2 * valid * hk * d + 2 * b * nk * hk * d) + 4 * b * h * nq
        return {"bytes": moved, "flops": 14 * pairs * h * d}
    if op == "lora":
        t, s, k, n, rank = _segments(case)[-1], case["requests"], case["k"], case["n"], case["rank"]
        used = min(s, case["adapters"])
        moved, flops = 2 * (t * k + 2 * case["tokens"] * n + used * rank * (k + n)), 2 * t * rank * (k + n)
        if case["train"]:  # dy read; dx, da, db written
            moved += 2 * (t * n + case["tokens"] * k + case["adapters"] * rank * (k + n))
            flops *= 3
        return {"bytes": moved, "flops": flops}
    b, n, d, rot = case["batch"], case["tokens"], case["dim"], case["rotary"]
    rows = b * n * (case["heads"] + case.get("kv_heads", 0))
    entry = 4 if case["table"] == "f32" else 2
    table = (b if case["positions"] else 1) * n * rot * entry
    if op == "rotate":
        return {"bytes": 4 * rows * d + table, "flops": 3 * rows * rot}
    passes = 4 if case["train"] else 2  # x read, y written; dy read, dx written
    return {"bytes": passes * 2 * rows * d + table, "flops": 5 * passes * rows * d}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "lora":
        return _exact_lora(case, s)
    cos, sin = _tables(s, torch.float64)
    if case["op"] == "rotate":
        return _exact_turn(s["x"].double(), cos, sin, case["layout"], 1.0)
    r = {}
    for name, weight, grad in (("q", "qw", "dq"), ("k", "kw", "dk")):
        x = s[name].double()
        w = torch.ones(case["dim"], device=DEV, dtype=torch.float64) if s[weight] is None else s[weight].double()
        rms = torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS)
        r[name] = _exact_turn(x / rms * w, cos, sin, case["layout"], 1.0)
        if case["train"]:
            back = _exact_turn(s[grad].double(), cos, sin, case["layout"], -1.0)
            r["d" + weight] = None if s[weight] is None else (back * x / rms).sum((0, 1, 2))
            along = (back * w * x).sum(-1, keepdim=True) / case["dim"]
            r[grad] = back * w / rms - x * along / rms ** 3
    return r


def _exact_turn(x, cos, sin, layout, sign):
    """Each pair of entries turned by its angle, as complex numbers."""
    half = cos.shape[-1]
    i = torch.arange(half, device=DEV)
    first, second = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
    z = torch.complex(x[..., first], x[..., second]) * torch.complex(cos, sign * sin)
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_attention(case, s):
    b, h, hk, d, nq, nk = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "nq", "nk"))
    f64 = {"device": DEV, "dtype": torch.float64}
    out, dq = torch.zeros(b, nq, h, d, **f64), torch.zeros(b, nq, h, d, **f64)
    dk, dv = torch.zeros(b, nk, hk, d, **f64), torch.zeros(b, nk, hk, d, **f64)
    lse = torch.full((b, h, nq), -math.inf, **f64)
    for i, n in enumerate(_key_lengths(case)):
        first = max(0, nq - n) if case["causal"] else 0  # queries before it see no key
        for j in range(h):
            g = j // (h // hk)
            q, do = s["q"][i, first:, j].double(), s["dout"][i, first:, j].double()
            k, v = s["k"][i, :n, g].double(), s["v"][i, :n, g].double()
            x = q @ k.t() / math.sqrt(d)
            if case["causal"]:
                x = x + torch.full_like(x, -math.inf).triu(1 + n - x.shape[0])
            z = torch.logsumexp(x, 1)
            p = torch.exp(x - z[:, None])
            dp = do @ v.t()
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(d)
            lse[i, j, first:], out[i, first:, j], dq[i, first:, j] = z, p @ v, ds @ k
            dk[i, :n, g] += ds.t() @ q
            dv[i, :n, g] += p.t() @ do
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _exact_lora(case, s):
    starts, ids = s["starts"].tolist(), s["ids"].tolist()
    y, dx = s["y"].double(), torch.zeros(case["tokens"], case["k"], device=DEV, dtype=torch.float64)
    da, db = torch.zeros_like(s["a"], dtype=torch.float64), torch.zeros_like(s["b"], dtype=torch.float64)
    for lo, hi, i in zip(starts, starts[1:], ids):
        x, a, b, f = s["x"][lo:hi].double(), s["a"][i].double(), s["b"][i].double(), s["scale"][i].double()
        low = x @ a.t()
        y[lo:hi] += f * (low @ b.t())
        if case["train"]:
            dy = s["dy"][lo:hi].double()
            dlow = f * (dy @ b)
            dx[lo:hi] = dlow @ a
            da[i] += dlow.t() @ x
            db[i] += f * (dy.t() @ low)
    return {"y": y, "dx": dx, "da": da, "db": db} if case["train"] else y
