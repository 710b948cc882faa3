"""The operators between a decoder block's products and at its end: what a pass of each is, its plain
form, and the cases it is measured at.

A decoder block of ``decode_ops`` keeps keys and values in 8 bits and weights in 4.  Around
the cache and the products it also needs

  heads    norms of queries and keys for each head, with the position rotation in the same pass
  gated    the first half of a gated feed-forward block: both projections with 4-bit weights, the
           activation and the product of the two
  sample   the next token from the logits: temperature, top-k, top-p and min-p, with given random numbers

``run`` computes them with elementary torch operations in 32 bits (64 where 32 lose what matters: the
angles of far positions, the masses of tokens next to a border), or, where ``own`` is true, through
the package's entry points.
"""
from __future__ import annotations

import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32,
          "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}
SIZE = {"bf16": 2, "fp16": 2, "f32": 4, "e4m3": 1, "int8": 1}
MASS = 45  # a token's mass is a whole number: 2^45 for the likeliest


def _ops():
    """The package (its folder's name is no identifier) and in it the operators."""
    name = "gemma4_omni_b200"
    if name not in sys.modules:
        folder = Path(__file__).resolve().parents[1] / "gemma-4-omni_b200"
        spec = importlib.util.spec_from_file_location(name, folder / "__init__.py",
                                                      submodule_search_locations=[str(folder)])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return importlib.import_module(name + ".decode_ops")


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one session's two soft tokens, a wide kv head: latency
        dict(name="heads-tick-2", op="heads", tokens=2, heads=8, kv_heads=1, dim=256, rotary=256, pairs="halves",
             base=10000.0, far=16384, dtype="bf16", weight="f32"),
        # answers of 64 sessions whose contexts are long, grouped kv heads
        dict(name="heads-answers-64", op="heads", tokens=64, heads=32, kv_heads=8, dim=128, rotary=128, pairs="halves",
             base=1000000.0, far=1000000, dtype="fp16", weight="same"),
        # the text histories of several sessions
        dict(name="heads-prompt", op="heads", tokens=16384, heads=32, kv_heads=8, dim=128, rotary=128, pairs="halves",
             base=10000.0, far=16384, dtype="bf16", weight="f32"),
        # the same in 32 bits, a quarter of each head rotated, neighbours paired
        dict(name="heads-partial-f32", op="heads", tokens=3001, heads=16, kv_heads=4, dim=64, rotary=16, pairs="neighbours",
             base=10000.0, far=16384, dtype="f32", weight="f32"),
        # one session's two soft tokens through the feed-forward block, 8-bit activations: latency
        dict(name="gated-tick-2", op="gated", rows=2, dim=1536, ffn=6144, group=128, x="e4m3", x_group=0,
             activation="silu", dtype="bf16"),
        # sixteen answers, 16-bit activations, finer groups
        dict(name="gated-answers-16", op="gated", rows=16, dim=2048, ffn=8192, group=64, x="bf16", x_group=0,
             activation="gelu", dtype="bf16"),
        # a tick of 250 sessions, int8 activations with scales for groups of columns, a ragged batch
        dict(name="gated-tick-500", op="gated", rows=499, dim=1536, ffn=6144, group=128, x="int8", x_group=128,
             activation="silu", dtype="bf16"),
        # text histories
        dict(name="gated-prompt", op="gated", rows=4096, dim=1536, ffn=6144, group=128, x="bf16", x_group=0,
             activation="silu", dtype="bf16"),
        # one session's next token, the usual filters: latency
        dict(name="sample-one", op="sample", rows=1, vocab=131072, dtype="bf16", temperature=0.8, top_k=64, top_p=0.95,
             min_p=0.0, per_row=False),
        # 64 answers, each session with settings of its own (greedy ones and ones without filters among them)
        dict(name="sample-answers-64", op="sample", rows=64, vocab=131072, dtype="bf16", temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.0, per_row=True),
        # 250 answers by their nucleus alone, 32-bit logits
        dict(name="sample-nucleus-250", op="sample", rows=250, vocab=131072, dtype="f32", temperature=1.0, top_k=0, top_p=0.9,
             min_p=0.0, per_row=False),
        # drafts of many sessions over a small, odd vocabulary
        dict(name="sample-drafts", op="sample", rows=1000, vocab=32003, dtype="fp16", temperature=0.7, top_k=0, top_p=1.0,
             min_p=0.05, per_row=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))


def draw(rng):
    op = rng.choice(["heads", "gated", "gated", "sample", "sample"])
    if op == "heads":
        dim = rng.choice([64, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 8])
        dtype = rng.choice(["bf16", "fp16", "f32"])
        most = 160_000_000 // ((heads + kv_heads) * dim * SIZE[dtype])
        return dict(op=op, tokens=_log(rng, 1, min(16384, most)), heads=heads, kv_heads=kv_heads, dim=dim,
                    rotary=rng.choice([dim, dim, dim // 2, dim // 4]), pairs=rng.choice(["halves", "halves", "neighbours"]),
                    base=rng.choice([10000.0, 500000.0, 1000000.0]), far=_log(rng, 1, 1000000), dtype=dtype,
                    weight=rng.choice(["f32", "same"]))
    if op == "gated":
        group = rng.choice([32, 64, 128])
        x = rng.choice(["bf16", "fp16", "e4m3", "int8"])
        dim = group * max(1, _log(rng, 128, 4096) // group)
        ffn = _log(rng, 64, min(16384, 33_000_000 // dim))
        rows = _log(rng, 1, min(4096, 30_000_000_000 // (dim * ffn)))
        x_group = 128 if x in TOP and dim % 128 == 0 and rng.random() < 0.4 else 0
        return dict(op=op, rows=rows, dim=dim, ffn=ffn, group=group, x=x, x_group=x_group,
                    activation=rng.choice(["silu", "gelu"]), dtype=rng.choice(["bf16", "fp16", "f32"]))
    vocab = _log(rng, 500, 262144)
    rows = _log(rng, 1, min(1000, 32_000_000 // vocab))
    return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["bf16", "fp16", "f32"]),
                temperature=rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]), top_k=rng.choice([0, 0, 1, _log(rng, 2, 5000)]),
                top_p=rng.choice([1.0, 0.95, 0.9, 0.5]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), per_row=rng.random() < 0.3)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    if op == "heads":
        # q and k are parts of one product's output: [tokens, heads + 2 kv_heads, dim]
        t, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        dt = DTYPES[case["dtype"]]
        both = (torch.randn(t, h + 2 * kv, d, generator=g, device="cuda") * 3.0).to(dt)
        q, k, _ = both.split((h, kv, kv), 1)
        w = [1.0 + 0.2 * torch.randn(d, generator=g, device="cuda") for _ in range(2)]
        if case["weight"] == "same":
            w = [v.to(dt) for v in w]
        at = torch.randint(0, case["far"], (t,), generator=g, device="cuda", dtype=torch.int32)
        s = dict(case=case, q=q, k=k, qw=w[0], kw=w[1], positions=at)
        if own:
            s["rotary"] = _ops().Rotary.create(d, rotary_dim=case["rotary"], base=case["base"], pairs=case["pairs"])
        return s
    if op == "gated":
        m, k, f = case["rows"], case["dim"], case["ffn"]
        codes = torch.randint(0, 256, (2 * f, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        scales = ((0.5 + torch.rand(2 * f, k // case["group"], generator=g, device="cuda")) * (0.25 * k ** -0.5)).to(torch.float16)
        x, xs = torch.randn(m, k, generator=g, device="cuda"), None
        if case["x"] in TOP:
            top = TOP[case["x"]]
            xg = x.view(m, -1, case["x_group"] or k)
            xs = xg.abs().amax(2) / top
            x = (xg / xs[:, :, None]).clamp(-top, top).view(m, k)
            x = x.round() if case["x"] == "int8" else x
        s = dict(case=case, x=x.to(DTYPES[case["x"]]), xs=xs, codes=codes, scales=scales)
        if own:
            s["weight"] = _ops().Int4Weight(codes, scales)
        return s
    # logits as a decoder leaves them: most tokens near one another, a few well above
    n, v = case["rows"], case["vocab"]
    x = torch.randn(n, v, generator=g, device="cuda") * 2.0
    few = min(40, v)
    step = v // few  # one in each part of the vocabulary: no index twice
    at = torch.arange(few, device="cuda") * step + torch.randint(0, step, (n, few), generator=g, device="cuda")
    ramp = 13.0 - 10.0 * torch.rand(n, few, generator=g, device="cuda") + torch.randn(n, few, generator=g, device="cuda")
    x.scatter_(1, at, ramp)
    s = dict(case=case, logits=x.to(DTYPES[case["dtype"]]), uniform=torch.rand(n, generator=g, device="cuda"))
    names = ("temperature", "top_k", "top_p", "min_p")
    if case["per_row"]:  # settings of the rows: the same set for every seed, in another order
        rng = random.Random(23)
        rows = [(rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]), rng.choice([0, 0, 20, 50, min(v, 400)]),
                 rng.choice([1.0, 0.95, 0.8]), rng.choice([0.0, 0.0, 0.05])) for _ in range(n)]
        random.Random(seed).shuffle(rows)
        for i, name in enumerate(names):
            s[name] = torch.tensor([r[i] for r in rows], dtype=torch.int32 if name == "top_k" else torch.float32, device="cuda")
    else:
        s.update({name: case[name] for name in names})
    return s


# ------------------------------------------------------------------ plain forms
def _rotate(x, cos, sin, rotary, pairs):
    """x [tokens, heads, dim], cos and sin [tokens, 1, rotary / 2]."""
    part, rest = x[..., :rotary], x[..., rotary:]
    if pairs == "halves":
        a, b = part[..., : rotary // 2], part[..., rotary // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_heads(s):
    c = s["case"]
    half = c["rotary"] // 2
    inv = c["base"] ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = s["positions"].double()[:, None, None] * inv
    cos, sin = angle.cos().float(), angle.sin().float()

    def side(x, w):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(2, keepdim=True) + 1e-6) * w.float()
        return _rotate(y, cos, sin, c["rotary"], c["pairs"]).to(x.dtype)

    return {"q": side(s["q"], s["qw"]), "k": side(s["k"], s["kw"])}


def _plain_gated(s):
    c = s["case"]
    m, k, f = c["rows"], c["dim"], c["ffn"]
    both = torch.stack([s["codes"] & 15, s["codes"] >> 4], 2).view(2 * f, k // c["group"], c["group"])
    w = ((both.float() - 8.0) * s["scales"].float()[:, :, None]).view(2 * f, k)
    x = s["x"].float()
    if s["xs"] is not None:
        x = (x.view(m, s["xs"].shape[1], -1) * s["xs"][:, :, None]).view(m, k)
    gate, up = torch.matmul(x, w.t()).split(f, 1)
    if c["activation"] == "silu":
        gate = gate / (1.0 + torch.exp(-gate))
    else:
        gate = 0.5 * gate * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate * gate * gate)))
    return {"out": (gate * up).to(DTYPES[c["dtype"]])}


def _column(value, n, dtype):
    if isinstance(value, torch.Tensor):
        return value.to(dtype)[:, None]
    return torch.full((n, 1), value, dtype=torch.float32, device="cuda").to(dtype)


def _plain_sample(s):
    c = s["case"]
    n, v = c["rows"], c["vocab"]
    heat, keep = _column(s["temperature"], n, torch.float64), _column(s["top_k"], n, torch.int64)
    top_p, min_p = _column(s["top_p"], n, torch.float64), _column(s["min_p"], n, torch.float64)
    x, order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)  # equal ones: the lower index first
    rank = torch.arange(v, device="cuda")
    x = x.double()
    mass = torch.exp((x - x[:, :1]) / torch.where(heat > 0, heat, 1.0))
    mass = torch.where((heat > 0) | (rank == 0), mass, 0.0)
    mass = torch.round(mass * 2.0 ** MASS).to(torch.int64)
    mass = torch.where((keep <= 0) | (rank < keep), mass, 0)
    whole = torch.cumsum(mass, 1)
    limit = torch.ceil(top_p * whole[:, -1:].double()).to(torch.int64).clamp(min=1)
    mass = torch.where((top_p >= 1.0) | (whole - mass < limit), mass, 0)
    mass = torch.where(mass >= torch.ceil(min_p * 2.0 ** MASS).to(torch.int64), mass, 0)
    mass = torch.zeros_like(mass).scatter_(1, order, mass)  # by index again
    upto = torch.cumsum(mass, 1)
    total = upto[:, -1:]
    target = torch.floor(s["uniform"].double()[:, None] * total.double()).to(torch.int64)
    target = torch.minimum(target, total - 1)
    token = torch.searchsorted(upto, target, right=True)
    logprob = torch.log(torch.gather(mass, 1, token).double() / total.double())
    return {"tokens": token[:, 0], "logprobs": logprob[:, 0].float()}


def run(s):
    c = s["case"]
    if own:
        ops = _ops()
        if c["op"] == "heads":
            q, k = ops.head_norm_rotary(s["q"], s["k"], s["positions"], s["rotary"], q_weight=s["qw"], k_weight=s["kw"], eps=1e-6)
            return {"q": q, "k": k}
        if c["op"] == "gated":
            return {"out": ops.w4_gated(s["x"], s["weight"], x_scale=s["xs"], activation=c["activation"],
                                        out_dtype=DTYPES[c["dtype"]])}
        tokens, logprobs = ops.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
                                             top_p=s["top_p"], min_p=s["min_p"], return_logprobs=True)
        return {"tokens": tokens, "logprobs": logprobs}
    return {"heads": _plain_heads, "gated": _plain_gated, "sample": _plain_sample}[c["op"]](s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "heads":
        size = SIZE[case["dtype"]]
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        weight = 4 if case["weight"] == "f32" else size
        return {"bytes": 2 * size * values + 4 * case["tokens"] + 2 * weight * case["dim"], "flops": 0}
    if case["op"] == "gated":
        m, k, f = case["rows"], case["dim"], case["ffn"]
        scales = 4 * m * (k // case["x_group"] if case["x_group"] else 1) if case["x"] in TOP else 0
        return {"bytes": f * k + 4 * f * (k // case["group"]) + m * k * SIZE[case["x"]] + scales + m * f * SIZE[case["dtype"]],
                "flops": 4 * m * k * f}
    n = case["rows"]
    return {"bytes": n * case["vocab"] * SIZE[case["dtype"]] + n * (4 + 8 + 4 + (16 if case["per_row"] else 0)), "flops": 0}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "heads":
        return _exact_heads(case, s)
    if case["op"] == "gated":
        return _exact_gated(case, s)
    return _exact_sample(case, s)


def _exact_heads(case, s):
    out, r = {}, case["rotary"]
    # a pair as one complex number, turned by its angle
    turns = torch.tensor([case["base"] ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float64, device="cuda")
    phase = torch.outer(s["positions"].double(), turns)
    phase = torch.polar(torch.ones_like(phase), phase)[:, None, :]
    for name in ("q", "k"):
        x = s[name].double()
        y = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["dim"] + 1e-6) * s[name + "w"].double()
        first = torch.arange(r // 2, device="cuda") * (1 if case["pairs"] == "halves" else 2)
        second = first + (r // 2 if case["pairs"] == "halves" else 1)
        z = torch.complex(y[..., first], y[..., second]) * phase
        y[..., first], y[..., second] = z.real, z.imag
        out[name] = y
    return out


def _exact_gated(case, s):
    f, k = case["ffn"], case["dim"]
    x = s["x"].double()
    if s["xs"] is not None:
        x = x * s["xs"].double().repeat_interleave(k // s["xs"].shape[1], 1)

    def product(rows):
        code = s["codes"][rows]
        w = torch.empty(code.shape[0], k, dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (code % 16).double() - 8, (code // 16).double() - 8
        return x @ (w * s["scales"][rows].double().repeat_interleave(case["group"], 1)).t()

    gate, up = product(slice(0, f)), product(slice(f, 2 * f))
    if case["activation"] == "silu":
        gate = gate * torch.sigmoid(gate)
    else:  # (1 + tanh z) / 2 = sigmoid(2 z)
        gate = gate * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate ** 3))
    return {"out": gate * up}


def _exact_sample(case, s):
    """Row by row, in the order of the definition; the tokens are whole numbers."""
    logprobs = torch.empty(case["rows"], dtype=torch.float64, device="cuda")
    index = torch.arange(case["vocab"], device="cuda")

    def setting(name, r):
        value = s[name]
        return value[r].double() if isinstance(value, torch.Tensor) else torch.tensor(value, dtype=torch.float32).double()

    for r in range(case["rows"]):
        x = s["logits"][r].double()
        heat, keep = float(setting("temperature", r)), int(setting("top_k", r))
        if heat == 0.0:
            logprobs[r] = 0.0
            continue
        order = torch.argsort(x, descending=True, stable=True)
        order = order[:keep] if keep > 0 else order
        mass = torch.round(2.0 ** MASS * torch.exp((x[order] - x[order[0]]) / heat)).to(torch.int64)
        p = float(setting("top_p", r))
        if p < 1.0:
            most = max(1, math.ceil(p * float(mass.sum())))
            first = int((torch.cumsum(mass, 0) < most).sum()) + 1
            order, mass = order[:first], mass[:first]
        live = mass >= math.ceil(float(setting("min_p", r)) * 2.0 ** MASS)
        order, mass = order[live], mass[live]
        back = torch.argsort(index[order])
        upto = torch.cumsum(mass[back], 0)
        total = int(upto[-1])
        target = min(total - 1, math.floor(float(s["uniform"][r].double()) * float(total)))
        chosen = int((upto <= target).sum())
        logprobs[r] = math.log(int(mass[back[chosen]]) / total)
    return {"tokens": None, "logprobs": logprobs}
