"""The text-decoder operators: what a pass of each is, its plain form, and the cases it is measured at.

The audio tower hands two soft tokens a session and tick to the text decoder.  The
decoder keeps a private, growing K/V cache for each session, in pages of 8-bit codes.
The operators are the ones a decoder block needs around that cache:

  plan     block tables and slot maps of a step, built on the GPU from the request lengths
  append   new keys and values written into the 8-bit cache (a scale per page and head)
  attend   attention over that cache
  norm     RMS norm with the residual's addition and an 8-bit output with scales
  w4       matrix-vector products with 4-bit weights and group scales

``run`` computes them with elementary torch operations in 32 bits, or, where ``own`` is
true, through the package's entry points.
"""
from __future__ import annotations

import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

F32 = torch.float32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32,
          "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}


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
        # a tick of a lightly loaded GPU: 16 sessions of 2 soft tokens each
        dict(name="plan-tick-16", op="plan", rows=16, sessions=64, pages=4096, page=64, max_pages=256,
             new="tick", new_max=2),
        # a tick of a full GPU: 2048 sessions, half of them with new tokens
        dict(name="plan-tick-2048", op="plan", rows=2048, sessions=4096, pages=262144, page=64, max_pages=256,
             new="tick", new_max=2),
        # the soft tokens of 128 sessions enter a cache with one wide kv head
        dict(name="append-tick-128", op="append", rows=128, new="tick", new_max=2, len_max=4096, kv_heads=1, dim=256,
             page=64, dtype="bf16"),
        # sixteen sessions are read in from their text history
        dict(name="append-prompt", op="append", rows=16, new="prompt", new_max=2048, len_max=1024, kv_heads=8, dim=128,
             page=32, dtype="bf16"),
        # one answer is written alone, at the longest context: latency
        dict(name="attend-one", op="attend", rows=1, new="answer", new_max=1, len_max=16384, heads=8, kv_heads=1,
             dim=256, page=64, window=0, softcap=0.0, dtype="bf16", ragged=False),
        # the soft tokens of 1024 sessions in a layer with a sliding window
        dict(name="attend-tick-1024", op="attend", rows=1024, new="tick", new_max=2, len_max=4096, heads=8, kv_heads=1,
             dim=256, page=64, window=1024, softcap=0.0, dtype="bf16", ragged=True),
        # 64 sessions write answers over ragged contexts with grouped kv heads
        dict(name="attend-answer-64", op="attend", rows=64, new="answer", new_max=1, len_max=16384, heads=32,
             kv_heads=8, dim=128, page=32, window=0, softcap=0.0, dtype="bf16", ragged=True),
        # sessions catch up after a pause: chunks of tokens against what is cached
        dict(name="attend-catch-up", op="attend", rows=8, new="prompt", new_max=512, len_max=8192, heads=16,
             kv_heads=4, dim=128, page=64, window=0, softcap=50.0, dtype="fp16", ragged=True),
        # two soft tokens of one session at the tower's width: latency
        dict(name="norm-tick-2", op="norm", rows=2, dim=1536, group=0, dtype="bf16", weight="f32", out="e4m3"),
        # the rows of several sessions' histories, scales for groups of 128 columns
        dict(name="norm-prompt", op="norm", rows=16384, dim=2048, group=128, dtype="bf16", weight="f32", out="e4m3"),
        # one session's two tokens through the first feed-forward matrix, 8-bit activations
        dict(name="w4-tick-2", op="w4", rows=2, out=6144, dim=1536, group=128, x="e4m3", x_group=0, dtype="bf16"),
        # sixteen answers through the vocabulary's matrix
        dict(name="w4-head-16", op="w4", rows=16, out=131072, dim=2048, group=64, x="bf16", x_group=0, dtype="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "norm", "w4"])
    if op == "plan":
        rows, page = _log(rng, 1, 2048), rng.choice([16, 32, 64, 128])
        kind = rng.choice(["tick", "tick", "prompt"])
        new_max = rng.choice([1, 2]) if kind == "tick" else _log(rng, 16, min(2048, max(16, 65536 // rows)))
        max_pages = _log(rng, 24 + 2048 // page, 320)
        return dict(op=op, rows=rows, sessions=rows + _log(rng, 1, 2048), pages=_log(rng, 4096 + 400 * rows // 4, 262144),
                    page=page, max_pages=max_pages, new=kind, new_max=new_max)
    if op == "append":
        kind = rng.choice(["tick", "answer", "prompt"])
        rows = _log(rng, 1, 16 if kind == "prompt" else 1024)
        dim = rng.choice([64, 128, 256])
        heads = rng.choice([1, 2, 4, 8]) if dim < 256 else rng.choice([1, 2, 4])
        return dict(op=op, rows=rows, new=kind, new_max={"tick": 2, "answer": 1}.get(kind) or _log(rng, 8, 2048),
                    len_max=_log(rng, 1, 1024 if rows > 64 else 4096), kv_heads=heads, dim=dim,
                    page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "fp16", "f32"]))
    if op == "attend":
        kind = rng.choice(["tick", "answer", "answer", "prompt"])
        dim = rng.choice([64, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8]) if dim < 256 else rng.choice([1, 2])
        heads = kv_heads * rng.choice([1, 2, 4, 8] if kv_heads < 8 else [1, 2, 4])
        rows = _log(rng, 1, 8 if kind == "prompt" else 1024)
        new_max = {"tick": 2, "answer": 1}.get(kind) or _log(rng, 8, 512)
        # what the plain form holds is bounded: keys of all rows, and scores
        most = min(16384, 550_000_000 // (rows * kv_heads * dim), 500_000_000 // (rows * heads * new_max))
        len_max = _log(rng, 1, max(2, most))
        return dict(op=op, rows=rows, new=kind, new_max=new_max, len_max=len_max, heads=heads, kv_heads=kv_heads, dim=dim,
                    page=rng.choice([16, 32, 64, 128]), window=rng.choice([0, 0, _log(rng, 1, 4096)]),
                    softcap=rng.choice([0.0, 0.0, 50.0]), dtype=rng.choice(["bf16", "fp16"]),
                    ragged=rng.random() < 0.8)
    if op == "norm":
        dim = 8 * _log(rng, 8, 1024) if rng.random() < 0.5 else _log(rng, 64, 8192)
        if dim == 3072:
            dim += 8
        group = rng.choice([0, 128])
        if group:
            dim = max(128, dim // 128 * 128)
            dim += 128 if dim == 3072 else 0
        return dict(op=op, rows=_log(rng, 1, max(1, 33_000_000 // dim)), dim=dim, group=group,
                    dtype=rng.choice(["bf16", "fp16", "f32"]), weight=rng.choice(["f32", "same"]), out="e4m3")
    group = rng.choice([32, 64, 128])
    dim = group * max(1, _log(rng, 128, 8192) // group)
    dim += group if dim == 3072 else 0
    out = _log(rng, 64, min(131072, 268_000_000 // dim))
    return dict(op=op, rows=_log(rng, 1, 16), out=out + (out == 3072), dim=dim, group=group,
                x=rng.choice(["bf16", "fp16", "e4m3", "int8"]), x_group=rng.choice([0, 128]) if dim % 128 == 0 else 0,
                dtype=rng.choice(["bf16", "fp16", "f32"]))


# ------------------------------------------------------------------ inputs
def _lengths(case, seed):
    """(tokens cached before the step, new tokens) of each row, as the mode has them.

    A case has the same set of rows for every seed, in another order: its outputs keep their shapes."""
    rng = random.Random(17)
    n, kind, top = case["rows"], case["new"], case["new_max"]
    if kind == "prompt":
        new = [rng.randint(max(1, top // 4), top) for _ in range(n)]
    elif kind == "tick":  # now and then a session has a single token, or none
        new = [top if rng.random() < 0.9 else rng.randint(0, top) for _ in range(n)]
    else:
        new = [1] * n
    if sum(new) == 0:
        new[0] = 1
    top = case.get("len_max") or case["page"] * case["max_pages"] - case["new_max"]
    if case["op"] == "plan":
        top = min(top, max(1, case["pages"] * case["page"] // (2 * n)))
    if case.get("ragged", True):
        old = [max(0, rng.randint(0, top) - m) if case["op"] == "attend" else rng.randint(0, top) for m in new]
    else:
        old = [max(0, top - m) for m in new]
    if case["op"] == "plan":
        old = [min(v, case["page"] * case["max_pages"] - m) for v, m in zip(old, new)]
    pairs = list(zip(old, new))
    random.Random(seed).shuffle(pairs)
    return [a for a, _ in pairs], [b for _, b in pairs]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _tables(lens, page, width, pages, g, slack=0):
    """Random distinct pages for rows of these lengths; -1 past a row's last page."""
    need = (_ints(lens) + page - 1) // page
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    first = torch.cumsum(need, 0) - need
    col = torch.arange(width, device="cuda")
    at = (first[:, None] + col).clamp(max=pages - 1)
    return torch.where(col < need[:, None], order[at], -1).to(torch.int32), order[: int(sum(-(-v // page) for v in lens))]


def _codes(shape, g):
    """8-bit codes as a quantiser leaves them: near normal, the largest at the end of the range."""
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat, step = out.view(-1), 1 << 28
    for a in range(0, flat.numel(), step):
        part = flat[a:a + step]
        part.copy_(torch.randn(part.numel(), generator=g, device="cuda").mul_(36.0).round_().clamp_(-127, 127))
    return out


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    if op == "plan":
        old, new = _lengths(case, seed)
        tabs, taken = _tables(old, case["page"], case["max_pages"], case["pages"], g)
        sessions = torch.randperm(case["sessions"], generator=g, device="cuda")[: case["rows"]].to(torch.int32)
        tables = torch.full((case["sessions"], case["max_pages"]), -1, dtype=torch.int32, device="cuda")
        lengths = torch.zeros(case["sessions"], dtype=torch.int32, device="cuda")
        tables[sessions.long()], lengths[sessions.long()] = tabs, _ints(old)
        words = -(-case["pages"] // 32)
        bits = torch.zeros(words * 32, dtype=torch.int64, device="cuda")
        bits[taken.long()] = 1
        used = (bits.view(words, 32) << torch.arange(32, device="cuda")).sum(1).to(torch.int32)
        s = dict(case=case, sessions=sessions, new=_ints(new), tables=tables, lengths=lengths, used=used, tokens=sum(new))
        if own:
            s["directory"] = _ops().PageDirectory(tables, lengths, used, pages=case["pages"], page_tokens=case["page"])
        return s
    if op in ("append", "attend"):
        old, new = _lengths(case, seed)
        page, h, d = case["page"], case["kv_heads"], case["dim"]
        lens = [a + b for a, b in zip(old, new)]
        used = sum(-(-v // page) for v in lens)
        pages = used + 3 + used // 16
        width = max(1, -(-max(lens) // page))
        tabs, taken = _tables(lens, page, width, pages, g)
        shape = (pages, h, page, d)
        kc, vc = _codes(shape, g), _codes(shape, g)
        # channels of keys differ more than those of values: their scales are larger; pages nobody has hold anything
        ks = torch.full((pages, h), float("nan"), device="cuda")
        vs = torch.full((pages, h), float("nan"), device="cuda")
        ks[taken.long()] = (0.5 + torch.rand(len(taken), h, generator=g, device="cuda")) * 6.0 / 127
        vs[taken.long()] = (0.5 + torch.rand(len(taken), h, generator=g, device="cuda")) * 3.5 / 127
        cu = torch.cat([_ints([0]), torch.cumsum(_ints(new), 0).to(torch.int32)])
        s = dict(case=case, kc=kc, vc=vc, ks=ks, vs=vs, tables=tabs, kv_len=_ints(lens), cu=cu, tokens=sum(new))
        if own:
            s["cache"] = _ops().Kv8Cache(kc, vc, ks, vs)
        if op == "append":
            t = torch.arange(s["tokens"], device="cuda")
            row = torch.searchsorted(cu[1:].long(), t, right=True)
            at = (_ints(old).long()[row] + t - cu.long()[row])
            s["slots"] = tabs.long()[row, at // page] * page + at % page
            dt = DTYPES[case["dtype"]]
            s["k"] = (torch.randn(s["tokens"], h, d, generator=g, device="cuda") * 1.5).to(dt)
            s["v"] = torch.randn(s["tokens"], h, d, generator=g, device="cuda").to(dt)
        else:
            s["q"] = torch.randn(s["tokens"], case["heads"], d, generator=g, device="cuda").to(DTYPES[case["dtype"]])
        return s
    if op == "norm":
        dt = DTYPES[case["dtype"]]
        m, d = case["rows"], case["dim"]
        x = torch.randn(m, d, generator=g, device="cuda").to(dt)
        r = (torch.randn(m, d, generator=g, device="cuda") * 4.0).to(dt)
        w = 1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")
        return dict(case=case, x=x, residual=r, weight=w if case["weight"] == "f32" else w.to(dt))
    m, k, o = case["rows"], case["dim"], case["out"]
    codes = torch.randint(0, 256, (o, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = ((0.5 + torch.rand(o, k // case["group"], generator=g, device="cuda")) * 0.01).to(torch.float16)
    x, xs = torch.randn(m, k, generator=g, device="cuda"), None
    if case["x"] in TOP:
        gx = case["x_group"] or k
        xg = x.view(m, k // gx, gx)
        xs = xg.abs().amax(2) / TOP[case["x"]]
        x = (xg / xs[:, :, None]).clamp(-TOP[case["x"]], TOP[case["x"]]).view(m, k)
        x = x.round() if case["x"] == "int8" else x
    s = dict(case=case, x=x.to(DTYPES[case["x"]]), xs=xs, codes=codes, scales=scales)
    if own:
        s["weight"] = _ops().Int4Weight(codes, scales)
    return s


# ------------------------------------------------------------------ plain forms
def _plain_plan(s):
    page, pages, width = s["case"]["page"], s["case"]["pages"], s["case"]["max_pages"]
    before = s["lengths"].long()[s["sessions"].long()]
    after = before + s["new"]
    p0, p1 = (before + page - 1) // page, (after + page - 1) // page
    rank = torch.cumsum(p1 - p0, 0) - (p1 - p0)
    bits = (s["used"][:, None] >> torch.arange(32, dtype=torch.int32, device="cuda")) & 1
    free = torch.nonzero(bits.view(-1)[:pages] == 0).view(-1)
    col = torch.arange(width, device="cuda")
    fresh = free[(rank[:, None] + col - p0[:, None]).clamp(0, free.numel() - 1)]
    rows = s["tables"].long()[s["sessions"].long()]
    rows = torch.where(col < p0[:, None], rows, torch.where(col < p1[:, None], fresh, -1))
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), torch.cumsum(s["new"].long(), 0)])
    t = torch.arange(s["tokens"], device="cuda")
    row = torch.searchsorted(cu[1:], t, right=True)
    at = before[row] + t - cu[row]
    slots = rows[row, at // page] * page + at % page
    return {"row_tables": rows.to(torch.int32), "kv_len": after.to(torch.int32), "cu_tokens": cu.to(torch.int32),
            "slots": slots, "positions": at.to(torch.int32), "token_rows": row.to(torch.int32)}


def _plain_append(codes, scale, x, slots, page):
    """One of the two sides of the cache, in place."""
    x = x.float()
    which, at = slots // page, slots % page
    touched, back = torch.unique(which, return_inverse=True)
    u, h = touched.numel(), x.shape[1]
    first = torch.full((u,), page, device="cuda").scatter_reduce_(0, back, at, "amin")
    fine = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs().amax(2)
    most = torch.zeros(u, h, device="cuda").scatter_reduce_(0, back[:, None].expand(-1, h), fine, "amax")
    s0 = torch.where(first[:, None] > 0, scale[touched], torch.zeros_like(most))
    s1 = torch.maximum(s0, most / torch.full_like(most, 127.0))
    held = codes[touched]
    again = torch.nan_to_num(torch.round(held.float() * s0[:, :, None, None] / s1[:, :, None, None]), nan=0.0)
    grown = (s1 != s0)[:, :, None, None] & (torch.arange(page, device="cuda") < first[:, None])[:, None, :, None]
    codes[touched] = torch.where(grown, again.clamp(-127, 127).to(torch.int8), held)
    new = torch.nan_to_num(torch.round(x / s1[back][:, :, None]), nan=0.0).clamp(-127, 127).to(torch.int8)
    codes[which, :, at] = new
    scale[touched] = s1


def _plain_attend(s):
    c, q = s["case"], s["q"].float()
    n, width = s["tables"].shape
    heads, kvh, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    length, top = width * page, c["new_max"]
    at = s["tables"].long().clamp(min=0)
    j = torch.arange(length, device="cuda")
    live = (j < s["kv_len"][:, None])[:, None, :, None]  # [n, 1, length, 1]

    def side(codes, scale):
        x = codes[at].float() * scale[at][..., None, None]
        return torch.where(live, x.permute(0, 2, 1, 3, 4).reshape(n, kvh, length, d), 0.0)

    new = s["cu"][1:] - s["cu"][:-1]
    i = torch.arange(top, device="cuda")
    token = (s["cu"][:-1, None] + i).clamp(max=s["tokens"] - 1).long()  # [n, top]
    here = i < new[:, None]
    pos = (s["kv_len"] - new)[:, None] + i
    qr = q[token].view(n, top, kvh, heads // kvh, d).permute(0, 2, 3, 1, 4).reshape(n, kvh, -1, d)
    x = torch.matmul(qr, side(s["kc"], s["ks"]).transpose(2, 3)).view(n, kvh, heads // kvh, top, length) / math.sqrt(d)
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    seen = here[:, :, None] & (j <= pos[:, :, None]) & (j < s["kv_len"][:, None, None])
    if c["window"]:
        seen &= j > pos[:, :, None] - c["window"]
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(4, keepdim=True)
    m = torch.where(torch.isinf(m), 0.0, m)
    p = torch.exp(x.sub_(m))
    total = p.sum(4, keepdim=True)
    y = torch.matmul(p.view(n, kvh, -1, length), side(s["vc"], s["vs"])).view(n, kvh, heads // kvh, top, d)
    y = torch.where(total > 0, y / total, 0.0)
    lse = (m + torch.log(total))[..., 0]
    y = y.permute(0, 3, 1, 2, 4).reshape(n, top, heads, d)[here]
    return {"out": y.to(s["q"].dtype), "lse": lse.permute(0, 3, 1, 2).reshape(n, top, heads)[here]}


def _plain_norm(s):
    c = s["case"]
    h = s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * s["weight"].float()
    y = y.view(c["rows"], -1, c["group"] or c["dim"])
    scale = y.abs().amax(2) / TOP[c["out"]]
    top = TOP[c["out"]]
    codes = torch.where(scale[:, :, None] > 0, y / scale[:, :, None], torch.zeros_like(y)).clamp(-top, top)
    return {"codes": codes.view(c["rows"], c["dim"]).to(DTYPES[c["out"]]), "scales": scale, "hidden": h.to(s["x"].dtype)}


def _plain_w4(s):
    c = s["case"]
    m, k, o = c["rows"], c["dim"], c["out"]
    both = torch.stack([s["codes"] & 15, s["codes"] >> 4], 2).view(o, k // c["group"], c["group"])
    w = ((both.float() - 8.0) * s["scales"].float()[:, :, None]).view(o, k)
    x = s["x"].float()
    if s["xs"] is not None:
        x = (x.view(m, s["xs"].shape[1], -1) * s["xs"][:, :, None]).view(m, k)
    return {"out": torch.matmul(x, w.t()).to(DTYPES[c["dtype"]])}


def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        ops = _ops()
        if op == "plan":
            p = s["directory"].plan(s["sessions"], s["new"], max_tokens=s["tokens"])
            return {"row_tables": p.row_tables, "kv_len": p.kv_len, "cu_tokens": p.cu_tokens, "slots": p.slots,
                    "positions": p.positions, "token_rows": p.token_rows}
        if op == "append":
            s["cache"].append(s["k"], s["v"], s["slots"])
            return {"k_codes": s["kc"], "v_codes": s["vc"], "k_scale": s["ks"], "v_scale": s["vs"]}
        if op == "attend":
            out, lse = ops.kv8_attention(s["q"], s["cache"], s["tables"], s["kv_len"], s["cu"], max_new=c["new_max"],
                                         window=c["window"], softcap=c["softcap"], return_lse=True)
            return {"out": out, "lse": lse}
        if op == "norm":
            codes, scales, hidden = ops.rms_norm8(s["x"], s["weight"], residual=s["residual"], eps=1e-6,
                                                  group=c["group"], dtype=DTYPES[c["out"]])
            return {"codes": codes, "scales": scales, "hidden": hidden}
        return {"out": ops.w4_matvec(s["x"], s["weight"], x_scale=s["xs"], out_dtype=DTYPES[c["dtype"]])}
    if op == "plan":
        return _plain_plan(s)
    if op == "append":
        _plain_append(s["kc"], s["ks"], s["k"], s["slots"], c["page"])
        _plain_append(s["vc"], s["vs"], s["v"], s["slots"], c["page"])
        return {"k_codes": s["kc"], "v_codes": s["vc"], "k_scale": s["ks"], "v_scale": s["vs"]}
    return {"attend": _plain_attend, "norm": _plain_norm, "w4": _plain_w4}[op](s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op, size = case["op"], {"bf16": 2, "fp16": 2, "f32": 4, "e4m3": 1, "int8": 1}
    if op in ("plan", "append", "attend"):
        old, new = _lengths(case, 1)
        t, page = sum(new), case["page"]
    if op == "plan":
        n = case["rows"]
        held = sum(-(-v // page) for v in old)
        return {"bytes": 12 * n + 4 * held + case["pages"] // 8 + 4 * n * case["max_pages"] + 8 * n + 4 + 16 * t, "flops": 0}
    if op == "append":
        h, d = case["kv_heads"], case["dim"]
        pages = sum(-(-(a + b) // page) - a // page for a, b in zip(old, new) if b)
        return {"bytes": 2 * t * h * d * (size[case["dtype"]] + 1) + 2 * 8 * pages * h + 8 * t, "flops": 0}
    if op == "attend":
        h, kvh, d, w = case["heads"], case["kv_heads"], case["dim"], case["window"]
        keys = pairs = 0
        for a, b in zip(old, new):
            if b:
                low = max(0, a + 1 - w) if w else 0
                keys += a + b - low
                if w:  # sum over the row's tokens of min(position + 1, w)
                    short = min(b, max(0, w - a))
                    pairs += short * a + short * (short + 1) // 2 + (b - short) * w
                else:
                    pairs += b * a + b * (b + 1) // 2
        return {"bytes": 2 * keys * kvh * d + 8 * (keys // page) * kvh + 4 * t * h * d + 4 * t * h,
                "flops": 4 * pairs * h * d}
    if op == "norm":
        m, d = case["rows"], case["dim"]
        return {"bytes": m * d * (3 * size[case["dtype"]] + 1) + 4 * m * (d // case["group"] if case["group"] else 1) + 4 * d,
                "flops": 0}
    m, k, o = case["rows"], case["dim"], case["out"]
    return {"bytes": o * k // 2 + 2 * o * (k // case["group"]) + m * k * size[case["x"]] + m * o * size[case["dtype"]],
            "flops": 2 * m * k * o}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    if op == "plan":
        return None  # whole numbers
    if op == "append":
        return _exact_append(case, s)
    if op == "norm":
        h = s["x"].double() + s["residual"].double()
        y = h / torch.sqrt(h.pow(2).sum(1, keepdim=True) / case["dim"] + 1e-6) * s["weight"].double()
        y = y.reshape(case["rows"], -1, case["group"] or case["dim"])
        scale = y.abs().amax(2) / TOP[case["out"]]
        codes = (y / scale[:, :, None]).reshape(case["rows"], case["dim"]).clamp(-448, 448)
        return {"codes": codes.to(DTYPES[case["out"]]).double(), "scales": scale, "hidden": h}
    if op == "w4":
        x = s["x"].double()
        if s["xs"] is not None:
            x = x * s["xs"].double().repeat_interleave(case["dim"] // s["xs"].shape[1], 1)
        parts = []
        for a in range(0, case["out"], 16384):
            code = s["codes"][a:a + 16384]
            w = torch.empty(code.shape[0], case["dim"], dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = (code % 16).double() - 8, (code // 16).double() - 8
            parts.append(x @ (w * s["scales"][a:a + 16384].double().repeat_interleave(case["group"], 1)).t())
        return {"out": torch.cat(parts, 1)}
    return _exact_attend(case, s)


def _exact_append(case, s):
    """The scales; the codes are whole numbers."""
    out, page, slots = {"k_codes": None, "v_codes": None}, case["page"], s["slots"]
    for name, x in (("k", s["k"]), ("v", s["v"])):
        scale = s[name + "s"].double()
        top = x.double().abs().amax(2) / 127.0
        fresh = torch.zeros_like(scale)
        where = slots // page
        starts = slots[slots % page == 0] // page  # a page that begins in this batch forgets its scale
        scale[starts] = 0.0
        fresh.index_reduce_(0, where, top, "amax")
        out[name + "_scale"] = torch.maximum(scale, fresh)
    return out


def _exact_attend(case, s):
    lens, cu = s["kv_len"].tolist(), s["cu"].tolist()
    heads, kvh, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(s["tokens"], heads, d, dtype=torch.float64, device="cuda")
    lse = torch.full((s["tokens"], heads), -math.inf, dtype=torch.float64, device="cuda")
    for r, n in enumerate(lens):
        a, b = cu[r], cu[r + 1]
        if b == a or n == 0:
            continue
        held = s["tables"][r, : -(-n // page)].long()
        k = (s["kc"][held].double() * s["ks"][held].double()[:, :, None, None]).transpose(0, 1).reshape(kvh, -1, d)[:, :n]
        v = (s["vc"][held].double() * s["vs"][held].double()[:, :, None, None]).transpose(0, 1).reshape(kvh, -1, d)[:, :n]
        q = s["q"][a:b].double().transpose(0, 1).reshape(kvh, heads // kvh * (b - a), d)
        x = (torch.bmm(q, k.transpose(1, 2)) * d ** -0.5).view(heads, b - a, n)
        if case["softcap"]:
            x = torch.tanh(x / case["softcap"]) * case["softcap"]
        pos = torch.arange(n - (b - a), n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        hidden = (key > pos) | ((key <= pos - case["window"]) if case["window"] else False)
        x.masked_fill_(hidden, -math.inf)
        total = torch.logsumexp(x, 2)
        p = torch.exp(x - total[:, :, None]).nan_to_num(0.0)
        y = torch.bmm(p.view(kvh, -1, n), v).view(heads, b - a, d)
        out[a:b], lse[a:b] = y.transpose(0, 1), total.t()
    return {"out": out, "lse": lse}
