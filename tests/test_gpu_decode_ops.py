"""The text-decoder operators against their definitions in 64 bits.

Bounds, from the arithmetic (u = half an ulp of the output's type, relative):
- page plans are whole numbers: equal.
- append: a code stands within half a step of its value; the division and the
  product before it are 32-bit, so 0.5 * scale * (1 + 1e-4); scales to 2 ulp.
- attention: a score is a sum of dim products in 32 bits, off by at most
  dx = dim * 2^-23 * scale * sum |q||k| (the softcap's tanh, within 4e-7 of its
  value, adds softcap * 4e-7); a probability is off by a factor 1 +- 2 dx (its own and
  the sum's) and by its rounding to 16 bits, 2^-11; so |out - ref| <= u |ref| +
  (2^-11 + 2 dx + 2^-18) sum p|v|, and lse is off by dx + 2^-20 (1 + |lse|).
- norm: the mean square and its root are good to 4e-6; a code is within half its
  format's step of y / scale.
- 4-bit products: k products summed in 32 bits, k * 2^-23 * sum |w||x|, and u |ref|.
"""
from __future__ import annotations

import math
import random

import pytest
import torch

from oracle import decode_ref

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3, I8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8
HALF_ULP = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


@pytest.fixture(scope="module")
def ops(pkg):
    from gemma4_omni_b200 import decode_ops
    return decode_ops


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ------------------------------------------------------------------ page plans
def random_directory(ops, rng, *, sessions, max_pages, pages, page):
    d = ops.PageDirectory.create(sessions=sessions, max_pages=max_pages, pages=pages, page_tokens=page)
    order = list(range(pages))
    rng.shuffle(order)
    tables = [[-1] * max_pages for _ in range(sessions)]
    lengths, used = [0] * sessions, [0] * pages
    for s in range(sessions):
        n = rng.choice([0, 0, 1, page - 1, page, page + 1, rng.randint(0, max_pages * page // 2)])
        held = -(-n // page)
        if held > len(order) // 2:
            continue
        lengths[s] = n
        for c in range(held):
            tables[s][c] = order.pop()
            used[tables[s][c]] = 1
    d.tables.copy_(torch.tensor(tables, dtype=torch.int32))
    d.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    words = [sum(1 << b for b in range(32) if 32 * w + b < pages and used[32 * w + b]) for w in range(-(-pages // 32))]
    d.used.copy_(torch.tensor([w - (1 << 32) if w >= 1 << 31 else w for w in words], dtype=torch.int32))
    return d, tables, lengths, used


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("rows,page,pages,new_max,seed", [
    (1, 16, 1, 1, 0), (1, 64, 33, 130, 1), (5, 16, 97, 40, 2), (40, 32, 1000, 3, 3), (300, 128, 4000, 2, 4),
    (1500, 16, 70001, 2, 5), (3, 256, 500, 20000, 6)])
def test_plan_and_commit_follow_the_page_rule(ops, rows, page, pages, new_max, seed):
    rng = random.Random(seed)
    sessions = rows + rng.randint(0, 7)
    d, tables, lengths, used = random_directory(ops, rng, sessions=sessions, max_pages=max(4, 2 * new_max // page + 3),
                                                pages=pages, page=page)
    for _ in range(3):
        who = rng.sample(range(sessions), rows)
        new = [rng.choice([0, 1, new_max, rng.randint(0, new_max)]) for _ in who]
        cap = sum(new) + rng.choice([1, 5])
        ref = decode_ref.plan(who, new, tables, lengths, used, page_tokens=page, max_tokens=cap)
        p = d.plan(ints(who), ints(new), max_tokens=cap)
        if ref is None:
            assert p.status() != 0
            d.commit(p)
            assert d.lengths.tolist() == lengths and d.tables.tolist() == tables
            continue
        row_tables, lens, slots, positions, owner = ref
        pad = [-1] * (cap - len(slots))
        assert p.status() == 0
        assert p.row_tables.tolist() == row_tables and p.kv_len.tolist() == lens
        assert p.slots.tolist() == slots + pad and p.positions.tolist() == positions + pad
        assert p.token_rows.tolist() == owner + pad
        assert p.cu_tokens.tolist() == [sum(new[:i]) for i in range(rows + 1)]
        d.commit(p)
        for s, t, n in zip(who, row_tables, lens):
            tables[s], lengths[s] = t, n
            for c in t:
                if c >= 0:
                    used[c] = 1
        assert d.lengths.tolist() == lengths and d.tables.tolist() == tables
        drop = who[: rows // 3]
        d.release(ints(drop))
        for s in drop:
            for c in tables[s]:
                if c >= 0:
                    used[c] = 0
            tables[s], lengths[s] = [-1] * len(tables[s]), 0
    assert d.status() == 0


def test_refused_plans_change_nothing(ops):
    d = ops.PageDirectory.create(sessions=4, max_pages=2, pages=3, page_tokens=16)
    for who, new, cap in [([1, 1], [1, 1], 8), ([0, 4], [1, 1], 8), ([-1], [1], 8), ([0], [-1], 8), ([0], [9], 8),
                          ([0], [33], 64), ([0, 1, 2], [17, 17, 1], 64)]:
        p = d.plan(ints(who), ints(new), max_tokens=cap)
        assert p.status() != 0
        assert set(p.slots.tolist()) == {-1} and set(p.kv_len.tolist()) == {0} and set(p.cu_tokens.tolist()) == {0}
        assert set(p.row_tables.flatten().tolist()) == {-1}
        d.commit(p)
    assert d.lengths.tolist() == [0] * 4 and d.used.tolist() == [0] and set(d.tables.flatten().tolist()) == {-1}
    d.release(ints([7]))
    assert d.status() != 0


# ------------------------------------------------------------------ append
def scatter_slots(rng, lens, new, page, pages):
    """Row tables over shuffled pages, and the slots of the new tokens in row order."""
    order = list(range(pages))
    rng.shuffle(order)
    tables = [[order.pop() for _ in range(-(-n // page))] for n in lens]
    slots = [t[p // page] * page + p % page for t, n, m in zip(tables, lens, new) for p in range(n - m, n)]
    return tables, slots


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim,heads,page,rows,new_max,layout,seed", [
    (64, 1, 16, 1, 1, "plain", 0), (256, 1, 64, 9, 2, "plain", 1), (128, 8, 32, 5, 100, "plain", 2),
    (64, 3, 128, 70, 2, "fused", 3), (128, 2, 256, 3, 700, "fused", 4), (128, 4, 16, 4, 33, "odd", 5)])
def test_append_keeps_one_scale_a_page(ops, dtype, dim, heads, page, rows, new_max, layout, seed):
    rng, g = random.Random(seed), gen(seed)
    cache = None
    lens = [0] * rows
    steps = [[rng.randint(0, new_max) for _ in range(rows)] for _ in range(3)]
    total = [sum(s[r] for s in steps) for r in range(rows)]
    pages = sum(-(-n // page) for n in total) + 2
    tables, _ = scatter_slots(rng, total, total, page, pages)
    cache = ops.Kv8Cache.create(pages=pages, kv_heads=heads, page_tokens=page, dim=dim)
    for name in ("k_scale", "v_scale"):
        getattr(cache, name).fill_(float("nan"))  # a page's first token forgets what the page had
    for step, new in enumerate(steps):
        slots = [tables[r][p // page] * page + p % page for r in range(rows) for p in range(lens[r], lens[r] + new[r])]
        n = len(slots)
        lens = [a + b for a, b in zip(lens, new)]
        if n == 0:
            continue
        raw = torch.randn(n, 2, heads, dim, generator=g, device="cuda") * (1.0 + step)  # the scales grow
        raw[rng.randrange(n)] = 0.0
        raw = raw.to(dtype)
        if layout == "odd":  # rows that are not 16-byte aligned
            wide = torch.zeros(n, 2, heads, dim + 1, dtype=dtype, device="cuda")
            wide[..., 1:] = raw
            k, v = wide[:, 0, :, 1:], wide[:, 1, :, 1:]
        else:  # "fused": strided views of one tensor
            k, v = (raw[:, 0], raw[:, 1]) if layout == "fused" else (raw[:, 0].contiguous(), raw[:, 1].contiguous())
        at = torch.tensor(slots + [-1], device="cuda")
        pad = lambda x: torch.cat([x, torch.full_like(x[:1], float("nan"))])  # noqa: E731  the padding token is skipped
        before = {s: (getattr(cache, s + "_codes").clone(), getattr(cache, s + "_scale").clone()) for s in "kv"}
        if layout == "plain":
            cache.append(pad(k), pad(v), at)
        else:
            cache.append(k, v, at[:-1])
        page_of, off = torch.div(at[:-1], page, rounding_mode="floor"), at[:-1] % page
        first = {}
        for s in slots:
            first[s // page] = min(first.get(s // page, page), s % page)
        for side, x in (("k", k), ("v", v)):
            codes, scale = getattr(cache, side + "_codes"), getattr(cache, side + "_scale")
            want = torch.where(torch.tensor([first.get(p, 1) == 0 for p in range(pages)], device="cuda")[:, None], 0.0,
                               before[side][1].double())
            want.index_reduce_(0, page_of, x.double().abs().amax(2) / 127, "amax")
            torch.testing.assert_close(scale.double(), want, rtol=2.0 ** -22, atol=1e-44, equal_nan=True)
            got = codes[page_of, :, off].double() * scale[page_of].double()[..., None]
            assert ((got - x.double()).abs() <= 0.5 * scale[page_of].double()[..., None] * (1 + 1e-4)).all()
            assert (codes >= -127).all()
            held, was = codes.clone(), before[side][0].clone()
            held[page_of, :, off], was[page_of, :, off] = 0, 0
            old = torch.tensor([[p in first and o < first[p] for o in range(page)] for p in range(pages)], device="cuda")
            old = old[:, None, :, None]
            grown = (scale != before[side][1])[:, :, None, None]
            assert torch.equal(torch.where(old & grown, 0, held), torch.where(old & grown, 0, was))
            drift = (held.double() * scale.double()[..., None, None] - was.double() * before[side][1].double()[..., None, None])
            assert (drift.abs() <= 0.5 * scale.double()[..., None, None] * (1 + 1e-4))[(old & grown).expand_as(held)].all()
    assert cache.status() == 0


def test_append_of_what_is_not_finite_and_of_bad_slots(ops, pkg):
    from gemma4_omni_b200 import _lib
    cache = ops.Kv8Cache.create(pages=2, kv_heads=1, page_tokens=16, dim=64)
    x = torch.linspace(-1, 1, 64, device="cuda").repeat(3, 1, 1).contiguous()
    x[0, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan])
    cache.append(x, torch.zeros_like(x), torch.tensor([16, 32, -5], device="cuda"))
    assert cache.k_codes[1, 0, 0, :4].tolist() == [127, -127, 0, round(float(x[0, 0, 3] / cache.k_scale[1, 0]))]
    assert abs(float(cache.k_scale[1, 0]) - 1 / 127) < 1e-8 and float(cache.v_scale[1, 0]) == 0.0
    assert not cache.v_codes.any() and not cache.k_codes[0].any()
    assert cache.status() == _lib.DEV_NONFINITE | _lib.DEV_BAD_PAGE


# ------------------------------------------------------------------ attention
def random_cache(ops, g, rng, lens, page, heads, dim):
    pages = sum(-(-n // page) for n in lens) + 2
    width = max(1, max(-(-n // page) for n in lens))
    tables, _ = scatter_slots(rng, lens, lens, page, pages)
    cache = ops.Kv8Cache.create(pages=pages, kv_heads=heads, page_tokens=page, dim=dim)
    # pages nobody reads, and codes past a row's end, hold anything
    for side in (cache.k_codes, cache.v_codes):
        side.copy_(torch.randint(-128, 128, side.shape, generator=g, device="cuda"))
    for side in (cache.k_scale, cache.v_scale):
        side.fill_(float("nan"))
        for t in tables:
            for p in t:
                side[p] = (0.2 + torch.rand(heads, generator=g, device="cuda")) * 3.0 / 127
    full = torch.full((len(lens), width), 2 ** 31 - 1, dtype=torch.int32)  # what is past a row's pages is not looked at
    for r, t in enumerate(tables):
        full[r, :len(t)] = torch.tensor(t, dtype=torch.int32)
    return cache, full.cuda()


def check_attention(ops, cache, tables, q, lens, cu, *, max_new, **how):
    kv_len, cut = ints(lens), ints(cu)
    out, lse = ops.kv8_attention(q, cache, tables, kv_len, cut, max_new=max_new, return_lse=True, **how)
    again = ops.kv8_attention(q, cache, tables, kv_len, cut, max_new=max_new, **how)
    assert torch.equal(out, again)  # nothing depends on the order in which parts finish
    dim = cache.dim
    scale = how.get("scale", dim ** -0.5)
    ref, ref_lse, spread, reach = decode_ref.attention(
        q, cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale, tables, kv_len, cut, scale=scale,
        window=how.get("window", 0), softcap=how.get("softcap", 0.0))
    dx = dim * 2.0 ** -23 * reach + 4e-7 * how.get("softcap", 0.0)
    bound = HALF_ULP[q.dtype] * ref.abs() + (2.0 ** -11 + 2 * dx[..., None] + 2.0 ** -18) * spread + 1e-7
    far = ((out.double() - ref).abs() / bound).max().item() if out.numel() else 0.0
    assert far <= 1.0, far
    empty = torch.isinf(ref_lse)
    assert torch.equal(empty, torch.isinf(lse)) and not out[empty].any()
    tol = dx + 2.0 ** -20 * (1 + ref_lse.abs())
    assert ((lse.double() - ref_lse).abs() <= tol)[~empty].all()
    assert cache.status() == 0


CASES = [  # dim, kv heads, group, page, lens, new, window, softcap
    (64, 1, 1, 16, [1], [1], 0, 0.0),
    (128, 1, 1, 64, [0, 1, 2, 15, 16, 17], [1, 1, 2, 1, 0, 1], 0, 0.0),
    (256, 1, 8, 64, [700, 64, 63, 65, 2, 1], [2, 2, 1, 2, 2, 1], 0, 0.0),
    (128, 8, 4, 32, [1000, 33, 257], [1, 1, 1], 0, 0.0),
    (64, 2, 3, 48, [500, 47, 49, 97], [1, 2, 3, 1], 0, 50.0),
    (128, 2, 16, 16, [300, 20], [3, 2], 17, 0.0),
    (256, 2, 1, 128, [3000, 5], [1, 1], 1000, 30.0),
    (128, 1, 8, 64, [5000], [1], 0, 0.0),
    (64, 4, 2, 256, [515, 260, 100], [130, 1, 100], 0, 0.0),
    (128, 2, 4, 64, [300, 90, 77], [65, 90, 3], 40, 50.0),
    (256, 1, 4, 32, [200, 400], [200, 31], 1, 0.0),
    (128, 1, 2, 16, [3, 0, 5], [7, 4, 9], 0, 0.0),  # more tokens than the cache holds: the first see nothing
    (64, 1, 5, 16, [1] * 40 + [900] + [0] * 9, [1] * 50, 0, 0.0),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention_against_64_bits(ops, dtype, case):
    dim, kvh, group, page, lens, new, window, softcap = CASES[case]
    rng, g = random.Random(case), gen(case)
    cache, tables = random_cache(ops, g, rng, [max(n, 1) for n in lens], page, kvh, dim)
    tokens = sum(new)
    q = torch.randn(tokens, kvh * group, dim, generator=g, device="cuda").to(dtype)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    check_attention(ops, cache, tables, q, lens, cu, max_new=max(new), window=window, softcap=softcap)


def test_attention_strides_padding_scale_and_range_of_q(ops):
    rng, g = random.Random(3), gen(3)
    cache, tables = random_cache(ops, g, rng, [130, 70], 32, 2, 128)
    wide = torch.randn(9, 3, 4, 128, generator=g, device="cuda").to(BF16)
    q = wide[:, 1]  # a slice of a fused projection
    q[2] *= 1e-20  # rows far from one another in range
    q[3] *= 60.0
    q[4, :, ::2] *= 1e-6
    check_attention(ops, cache, tables, q, [130, 70], [0, 4, 7], max_new=4, scale=0.03)
    out, lse = ops.kv8_attention(q, cache, tables, ints([130, 70]), ints([0, 4, 7]), max_new=4, return_lse=True)
    assert not out[7:].any() and torch.isinf(lse[7:]).all()  # tokens of no row


def test_attention_with_heavy_and_with_equal_scores(ops):
    rng, g = random.Random(4), gen(4)
    cache, tables = random_cache(ops, g, rng, [900], 64, 1, 64)
    q = torch.randn(2, 4, 64, generator=g, device="cuda")
    q[0, 0] = 0.0   # every key counts the same
    q[0, 1] *= 500.0  # one key counts alone
    check_attention(ops, cache, tables, q.to(F16), [900], [0, 2], max_new=2)


def test_attention_of_a_zero_scale_and_of_a_bad_page(ops, pkg):
    from gemma4_omni_b200 import _lib
    rng, g = random.Random(5), gen(5)
    cache, tables = random_cache(ops, g, rng, [64], 16, 1, 64)
    cache.v_scale[tables[0, 1]] = 0.0
    cache.k_scale[tables[0, 2]] = 0.0
    q = torch.randn(1, 2, 64, generator=g, device="cuda").to(BF16)
    check_attention(ops, cache, tables, q, [64], [0, 1], max_new=1)
    tables[0, 3] = -1
    out = ops.kv8_attention(q, cache, tables, ints([64]), ints([0, 1]), max_new=1)
    assert cache.status() == _lib.DEV_BAD_PAGE
    cache.status_word.zero_()
    pos = ops.kv8_attention(q, cache, tables, ints([48]), ints([0, 1]), max_new=1)
    torch.testing.assert_close(out, pos, rtol=0, atol=2 ** -7)


def test_attention_reads_a_cache_past_32_bits(ops):
    page, dim, heads = 256, 256, 8
    pages = (2 ** 31 + 2 ** 28) // (page * dim * heads)  # codes past 2^31 bytes
    cache = ops.Kv8Cache.create(pages=pages, kv_heads=heads, page_tokens=page, dim=dim)
    g = gen(6)
    k = torch.randn(300, heads, dim, generator=g, device="cuda").to(BF16)
    v = torch.randn(300, heads, dim, generator=g, device="cuda").to(BF16)
    tables = ints([[pages - 1, pages - 3]])
    slots = torch.tensor([int(tables[0, i // page]) * page + i % page for i in range(300)], device="cuda")
    cache.append(k, v, slots)
    q = torch.randn(1, heads, dim, generator=g, device="cuda").to(BF16)
    check_attention(ops, cache, tables, q, [300], [0, 1], max_new=1)


# ------------------------------------------------------------------ norm
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("out", [E4M3, I8])
@pytest.mark.parametrize("rows,dim,group,plain_weight", [
    (1, 1, 0, True), (2, 1536, 0, True), (3, 65, 0, False), (5, 2048, 128, True), (1, 16384, 0, True), (33, 200, 40, False),
    (7, 1000, 8, True), (300, 128, 128, False), (4, 4099, 0, True)])
def test_norm_codes_and_scales(ops, dtype, out, rows, dim, group, plain_weight):
    g = gen(rows + dim)
    wide = torch.randn(rows, 2, dim + 3, generator=g, device="cuda").to(dtype)
    x, res = wide[:, 0, :dim], wide[:, 1, 3:]
    w = 1 + 0.3 * torch.randn(dim, generator=g, device="cuda")
    w = w if plain_weight else w.to(dtype)
    codes, scales, hidden = ops.rms_norm8(x, w, residual=res, eps=1e-5, group=group, dtype=out)
    h, y = decode_ref.rms_norm(x, res, w, eps=1e-5)
    assert ((hidden.double() - h).abs() <= HALF_ULP[dtype] * (1 + 1e-3) * h.abs() + 1e-9).all()
    y = y.view(rows, -1, group or dim)
    top = 448 if out is E4M3 else 127
    want = y.abs().amax(2) / top
    assert codes.dtype is out and scales.shape == want.shape
    torch.testing.assert_close(scales.double(), want, rtol=4e-6, atol=1e-44)
    s = want[..., None]
    near = 0.5 * s if out is I8 else torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * s)
    got = codes.double().view(y.shape) * scales.double()[..., None]
    assert ((got - y).abs() <= near * (1 + 1e-3) + 1e-5 * y.abs()).all()


def test_norm_of_zero_rows_nan_and_no_residual(ops):
    x = torch.randn(4, 256, generator=gen(1), device="cuda").to(BF16)
    x[1] = 0.0
    x[2, 5] = math.nan
    x[3, 200] = math.inf
    for out in (E4M3, I8):
        codes, scales, hidden = ops.rms_norm8(x, torch.ones(256, device="cuda"), group=128, dtype=out)
        assert hidden is x and not codes[1].float().any() and scales[1].tolist() == [0.0, 0.0]
        assert torch.isnan(scales[2]).all() and not codes[2].float().any()
        assert scales[3, 0] == 0.0 and torch.isnan(scales[3, 1])
        _, y = decode_ref.rms_norm(x[:1], None, torch.ones(256, device="cuda"), eps=1e-6)
        torch.testing.assert_close(scales[:1].double(), y.abs().view(1, 2, 128).amax(2) / (448 if out is E4M3 else 127),
                                   rtol=4e-6, atol=0)


# ------------------------------------------------------------------ 4-bit products
@pytest.mark.parametrize("kind,x_group", [(BF16, 0), (F16, 0), (E4M3, 0), (E4M3, 128), (I8, 0), (I8, 256)])
@pytest.mark.parametrize("rows,out,k,group,out_dtype", [
    (1, 1, 256, 32, F32), (1, 2048, 1536, 128, BF16), (2, 6144, 1536, 128, F32), (3, 100, 512, 64, F16), (8, 257, 768, 32, F32),
    (9, 33, 2048, 128, BF16), (16, 4097, 256, 64, F32), (37, 70, 1024, 32, F32), (1, 515, 8192, 128, F32)])
def test_w4_products(ops, kind, x_group, rows, out, k, group, out_dtype):
    g = gen(rows + out)
    codes = torch.randint(0, 256, (out, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.01 * (0.1 + torch.rand(out, k // group, generator=g, device="cuda"))).to(F16)
    weight = ops.Int4Weight(codes, scales)
    x, xs = torch.randn(rows, k + 16, generator=g, device="cuda"), None
    if kind in (E4M3, I8):
        x, xs, _ = ops.rms_norm8(x[:, :k], torch.ones(k, device="cuda"), group=x_group, dtype=kind)
    else:
        x = x.to(kind)[:, 8:k + 8]
        x[0, :4] *= 2.0 ** -12 if kind is F16 else 2.0 ** -60
    y = ops.w4_matvec(x, weight, x_scale=xs, out_dtype=out_dtype)
    ref, spread = decode_ref.w4_product(x, xs, codes, scales)
    assert y.dtype is out_dtype and tuple(y.shape) == (rows, out)
    bound = HALF_ULP[out_dtype] * (1 + 1e-3) * ref.abs() + k * 2.0 ** -23 * spread + 1e-9
    assert ((y.double() - ref).abs() <= bound).all()
    wide = torch.zeros(rows, out + 5, dtype=out_dtype, device="cuda")
    ops.w4_matvec(x, weight, x_scale=xs, out=wide[:, 2:out + 2])
    assert torch.equal(wide[:, 2:out + 2], y) and not wide[:, :2].any() and not wide[:, out + 2:].any()


def test_w4_group_of_one_k_block_and_quantize(ops):
    w = torch.randn(40, 96, generator=gen(2), device="cuda")
    q = ops.Int4Weight.quantize(w, group=32)
    s = q.scales.float().repeat_interleave(32, 1)
    assert ((q.dequantize() - w).abs() <= 0.5 * s * (1 + 1e-2) + 1e-6).all()
    x = torch.randn(5, 96, generator=gen(3), device="cuda").to(BF16)
    ref, spread = decode_ref.w4_product(x, None, q.codes, q.scales)
    y = ops.w4_matvec(x, q, out_dtype=F32)
    assert ((y.double() - ref).abs() <= 96 * 2.0 ** -23 * spread + 2.0 ** -23 * ref.abs()).all()


def test_w4_nan_rows_stay_nan(ops):
    q = ops.Int4Weight.quantize(torch.randn(32, 256, generator=gen(4), device="cuda"))
    x = torch.zeros(2, 256, device="cuda").to(BF16)
    x[1, 7] = math.nan
    y = ops.w4_matvec(x, q)
    assert not y[0].any() and torch.isnan(y[1]).all()


# ------------------------------------------------------------------ streams, graphs, refusals
def test_calls_run_on_the_current_stream_and_in_graphs(ops):
    rng, g = random.Random(8), gen(8)
    cache, tables = random_cache(ops, g, rng, [200, 70], 32, 2, 128)
    q = torch.randn(2, 8, 128, generator=g, device="cuda").to(BF16)
    weight = ops.Int4Weight.quantize(torch.randn(256, 1024, generator=g, device="cuda"))
    ones = torch.ones(1024, device="cuda")
    kv_len, cu = ints([200, 70]), ints([0, 1, 2])

    def chain():
        y = ops.kv8_attention(q, cache, tables, kv_len, cu, max_new=1).view(2, 1024)
        codes, scales, _ = ops.rms_norm8(y, ones, residual=y)
        return ops.w4_matvec(codes, weight, x_scale=scales)

    want = chain()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain()
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = chain()
    q.copy_(torch.randn(2, 8, 128, generator=g, device="cuda"))
    kv_len.copy_(ints([150, 33]))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, chain())


def test_refusals(ops):
    cache = ops.Kv8Cache.create(pages=2, kv_heads=2, page_tokens=16, dim=64)
    x = torch.zeros(3, 2, 64, device="cuda")
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    one, cu = ints([1]), ints([0, 1])
    tables = ints([[0]])
    q = torch.zeros(1, 4, 64, device="cuda").to(BF16)
    d = ops.PageDirectory.create(sessions=2, max_pages=2, pages=4, page_tokens=16)
    w = ops.Int4Weight.quantize(torch.zeros(8, 128, device="cuda"))
    ones = torch.ones(128, device="cuda")
    bad = [
        lambda: ops.Kv8Cache.create(pages=2, kv_heads=2, page_tokens=24, dim=64),
        lambda: ops.Kv8Cache.create(pages=2, kv_heads=2, page_tokens=16, dim=80),
        lambda: ops.Kv8Cache.create(pages=2, kv_heads=2, page_tokens=16, dim=64, device="cpu"),
        lambda: cache.append(x, x.half(), slots),
        lambda: cache.append(x, x, slots[:2]),
        lambda: cache.append(x, x, slots.int()),
        lambda: cache.append(x.transpose(1, 2).contiguous().transpose(1, 2), x, slots),
        lambda: cache.append(x.int(), x.int(), slots),
        lambda: ops.kv8_attention(q.float(), cache, tables, one, cu, max_new=1),
        lambda: ops.kv8_attention(q[:, :3], cache, tables, one, cu, max_new=1),
        lambda: ops.kv8_attention(q, cache, tables, one.long(), cu, max_new=1),
        lambda: ops.kv8_attention(q, cache, tables, one, cu[:1], max_new=1),
        lambda: ops.kv8_attention(q, cache, tables, one, cu, max_new=1, window=-1),
        lambda: ops.kv8_attention(q, cache, tables, one, cu, max_new=0),
        lambda: ops.kv8_attention(q, cache, tables, one, cu, max_new=1, out=torch.zeros_like(q.float())),
        lambda: d.plan(ints([0, 1]), ints([1]), max_tokens=4),
        lambda: d.plan(ints([0]), ints([1]), max_tokens=0),
        lambda: d.plan(torch.zeros(1, dtype=torch.int64, device="cuda"), ints([1]), max_tokens=4),
        lambda: ops.PageDirectory.create(sessions=2, max_pages=2, pages=4, page_tokens=20),
        lambda: ops.rms_norm8(torch.zeros(2, 128, device="cuda"), ones[:64]),
        lambda: ops.rms_norm8(torch.zeros(2, 128, device="cuda"), ones, group=100),
        lambda: ops.rms_norm8(torch.zeros(2, 128, device="cuda"), ones, dtype=torch.uint8),
        lambda: ops.rms_norm8(torch.zeros(2, 128, device="cuda"), ones, residual=torch.zeros(2, 64, device="cuda")),
        lambda: ops.w4_matvec(torch.zeros(2, 128, device="cuda"), w),
        lambda: ops.w4_matvec(torch.zeros(2, 64, device="cuda").to(BF16), w),
        lambda: ops.w4_matvec(torch.zeros(2, 128, device="cuda").to(I8), w),
        lambda: ops.w4_matvec(torch.zeros(2, 128, device="cuda").to(BF16), w, out_dtype=torch.int32),
        lambda: ops.Int4Weight(w.codes, w.scales.float()),
        lambda: ops.Int4Weight(w.codes[:, :50], w.scales),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was accepted")
    # nothing to do is no error
    assert ops.kv8_attention(q[:0], cache, tables, one, ints([0, 0]), max_new=1).shape == (0, 4, 64)
    assert ops.w4_matvec(torch.zeros(0, 128, device="cuda").to(BF16), w).shape == (0, 8)
    assert ops.rms_norm8(torch.zeros(0, 128, device="cuda"), ones)[0].shape == (0, 128)
    cache.append(x[:0], x[:0], slots[:0])


# ------------------------------------------------------------------ the paths that sizes choose
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,dim,group", [(1184, 8, 0), (1200, 256, 128), (2000, 512, 0), (1300, 1024, 64), (1190, 2048, 128),
                                            (1185, 2056, 8), (1200, 4096, 256), (1184, 8192, 0), (1200, 16384, 128)])
def test_norm_with_a_row_for_every_scheduler(ops, dtype, rows, dim, group):
    g = gen(rows + dim)
    x = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
    res = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
    w = 1 + 0.3 * torch.randn(dim, generator=g, device="cuda")
    for out in (E4M3, I8):
        codes, scales, hidden = ops.rms_norm8(x, w, residual=res, group=group, dtype=out)
        h, y = decode_ref.rms_norm(x, res, w, eps=1e-6)
        assert ((hidden.double() - h).abs() <= HALF_ULP[dtype] * (1 + 1e-3) * h.abs() + 1e-9).all()
        y = y.view(rows, -1, group or dim)
        want = y.abs().amax(2) / (448 if out is E4M3 else 127)
        torch.testing.assert_close(scales.double(), want, rtol=4e-6, atol=1e-44)
        s = want[..., None]
        near = 0.5 * s if out is I8 else torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * s)
        got = codes.double().view(y.shape) * scales.double()[..., None]
        assert ((got - y).abs() <= near * (1 + 1e-3) + 1e-5 * y.abs()).all()


def test_norm_of_values_near_the_ends_of_the_range(ops):
    x = torch.randn(3, 256, generator=gen(11), device="cuda")
    x[1] *= 1e-30  # with eps the row is tiny: its scale is far below 2^-100
    x[2] *= 1e15
    codes, scales, _ = ops.rms_norm8(x, torch.full((256,), 1e-3, device="cuda"), eps=1e-6, dtype=I8)
    _, y = decode_ref.rms_norm(x, None, torch.full((256,), 1e-3, device="cuda"), eps=1e-6)
    got = codes.double() * scales.double()
    assert ((got - y).abs() <= 0.5 * scales.double() * (1 + 1e-3) + 1e-5 * y.abs()).all()


@pytest.mark.parametrize("rows,out,k,kind", [(16, 20000, 256, BF16), (1, 40000, 128, F16), (16, 160, 8192, BF16), (7, 64, 16384, F16),
                                             (12, 96, 16384, I8), (2, 4700, 1024, E4M3), (33, 9000, 512, BF16)])
def test_w4_products_in_every_arrangement(ops, rows, out, k, kind):
    g = gen(out + k)
    codes = torch.randint(0, 256, (out, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.01 * (0.1 + torch.rand(out, k // 64, generator=g, device="cuda"))).to(F16)
    weight = ops.Int4Weight(codes, scales)
    x, xs = torch.randn(rows, k, generator=g, device="cuda"), None
    if kind in (E4M3, I8):
        x, xs, _ = ops.rms_norm8(x, torch.ones(k, device="cuda"), dtype=kind)
    else:
        x = x.to(kind)
    y = ops.w4_matvec(x, weight, x_scale=xs, out_dtype=F32)
    ref, spread = decode_ref.w4_product(x, xs, codes, scales)
    assert ((y.double() - ref).abs() <= k * 2.0 ** -23 * spread + 2.0 ** -23 * ref.abs() + 1e-9).all()


@pytest.mark.parametrize("rows,lens,new", [(700, 40, 1), (300, 5, 2), (1, 16300, 1), (2, 9000, 40)])
def test_attention_over_many_rows_and_long_ones(ops, rows, lens, new):
    rng, g = random.Random(rows), gen(rows)
    n = [rng.randint(new, lens) if rows > 2 else lens for _ in range(rows)]
    cache, tables = random_cache(ops, g, rng, n, 64, 1, 128)
    q = torch.randn(rows * new, 8, 128, generator=g, device="cuda").to(F16)
    check_attention(ops, cache, tables, q, n, [new * i for i in range(rows + 1)], max_new=new)


def test_attention_scale_signs_and_inputs_that_are_not_finite(ops):
    rng, g = random.Random(12), gen(12)
    cache, tables = random_cache(ops, g, rng, [200], 32, 1, 64)
    q = torch.randn(1, 4, 64, generator=g, device="cuda").to(BF16)
    check_attention(ops, cache, tables, -q, [200], [0, 1], max_new=1, scale=0.2)
    plain = ops.kv8_attention(-q, cache, tables, ints([200]), ints([0, 1]), max_new=1, scale=0.2)
    turned = ops.kv8_attention(q, cache, tables, ints([200]), ints([0, 1]), max_new=1, scale=-0.2)
    torch.testing.assert_close(turned, plain, rtol=2 ** -7, atol=1e-3)  # the same scores: one store's rounding
    q[0, 1, 5], q[0, 2, 6] = math.nan, math.inf
    out, lse = ops.kv8_attention(q, cache, tables, ints([200]), ints([0, 1]), max_new=1, return_lse=True)
    assert torch.isnan(out[0, 1:3]).all() and torch.isnan(lse[0, 1:3]).all()
    assert torch.isfinite(out[0, [0, 3]]).all() and torch.isfinite(lse[0, [0, 3]]).all()


@pytest.mark.parametrize("dim,page,tokens", [(256, 128, 300), (128, 256, 700), (80, 16, 50)])
def test_append_of_groups_larger_than_the_registers_hold(ops, pkg, dim, page, tokens):
    """Through the C entry too, whose dim may be any multiple of 16."""
    from gemma4_omni_b200 import _lib
    g = gen(dim)
    pages = -(-tokens // page)
    kc, vc = (torch.zeros(pages, 2, page, dim, dtype=I8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages, 2, device="cuda") for _ in range(2))
    k, v = (torch.randn(tokens, 2, dim, generator=g, device="cuda") for _ in range(2))
    slots = torch.arange(tokens, device="cuda")
    _lib.check("lb_op_kv8_append", _lib.load().lb_op_kv8_append(
        k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), _lib.LB_F32, tokens, 2, dim, slots.data_ptr(),
        kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, page, None, torch.cuda.current_stream().cuda_stream))
    for codes, scale, x in ((kc, ks, k), (vc, vs, v)):
        got = (codes.double() * scale.double()[..., None, None]).transpose(1, 2).reshape(-1, 2, dim)[:tokens]
        step = scale.double().repeat_interleave(page, 0)[:tokens, :, None]
        assert ((got - x.double()).abs() <= 0.5 * step * (1 + 1e-4)).all()
        top = torch.stack([x[p * page:(p + 1) * page].double().abs().amax((0, 2)) for p in range(pages)]) / 127
        torch.testing.assert_close(scale.double(), top, rtol=2.0 ** -22, atol=0)


@pytest.mark.parametrize("rows,dim,group", [(1500, 100, 0), (1184, 999, 27), (1300, 1020, 12), (1200, 1027, 0), (5, 14001, 0), (1191, 320, 40)])
def test_norm_of_odd_widths_in_many_rows(ops, rows, dim, group):
    g = gen(rows + dim)
    for dtype in (BF16, F32):
        x, res = (torch.randn(rows, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
        x[1] = 0.0
        res[1] = 0.0
        w = 1 + 0.3 * torch.randn(dim, generator=g, device="cuda")
        codes, scales, hidden = ops.rms_norm8(x, w, residual=res, group=group, dtype=I8)
        h, y = decode_ref.rms_norm(x, res, w, eps=1e-6)
        assert ((hidden.double() - h).abs() <= HALF_ULP[dtype] * (1 + 1e-3) * h.abs() + 1e-9).all()
        y = y.view(rows, -1, group or dim)
        want = y.abs().amax(2) / 127
        torch.testing.assert_close(scales.double(), want, rtol=4e-6, atol=1e-44)
        got = codes.double().view(y.shape) * scales.double()[..., None]
        assert ((got - y).abs() <= 0.5 * want[..., None] * (1 + 1e-3) + 1e-5 * y.abs()).all()


def test_exchanged_tensors_of_directory_and_cache_are_followed(ops):
    pages = ops.PageDirectory.create(sessions=2, max_pages=4, pages=8, page_tokens=16)
    cache = ops.Kv8Cache.create(pages=8, kv_heads=1, page_tokens=16, dim=64)
    old = (pages.tables, pages.lengths, pages.used, cache.k_codes, cache.k_scale)
    before = [t.clone() for t in old]
    pages.tables, pages.lengths, pages.used = (t.clone() for t in old[:3])
    cache.k_codes, cache.k_scale = old[3].clone(), old[4].clone()
    pages.lengths[1] = 5
    pages.tables[1, 0] = 3
    pages.used[0] = 1 << 3
    ids = torch.tensor([1], dtype=torch.int32, device="cuda")
    plan = pages.plan(ids, torch.full_like(ids, 2), max_tokens=2)
    assert plan.status() == 0 and plan.kv_len.tolist() == [7] and plan.slots.tolist() == [3 * 16 + 5, 3 * 16 + 6]
    k = torch.ones(2, 1, 64, device="cuda")
    cache.append(k, k, plan.slots)
    pages.commit(plan)
    assert cache.k_codes[3, 0, 5:7].eq(127).all() and pages.lengths.tolist() == [0, 7]
    assert all(torch.equal(a, b) for a, b in zip(old, before))
