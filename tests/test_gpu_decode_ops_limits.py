"""The text-decoder operators where their inputs' ranges and contracts end.

Attention's bound, from what the kernel holds (all relative to one query):
- q is rounded to 2^-30 of its row's largest value, the sums of products are joined in 32 bits:
  a score is off by dx <= 2^-30 * scale * max|q| * sum |k| + 2^-21 * scale * sum |q||k|
  + 2^-21 (1 + |score|) (the exponential's argument and its approximation);
- p * sv is rounded to a step of 1 / (63 * 2^16) of the largest p * sv among the tile's keys that the query
  sees: half a step times sum |code| of the tile's keys;
- a capped score is off by 2^-19 of itself beside that;
- factors, the sum of p and the division: 2^-20 of sum p|v|;
- the output's half ulp (and its smallest step).
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
SMALLEST = {BF16: 2.0 ** -133, F16: 2.0 ** -25}


@pytest.fixture(scope="module")
def ops(pkg):
    from gemma4_omni_b200 import decode_ops
    return decode_ops


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make_cache(ops, g, lens, page, heads, dim):
    """Random codes and scales on shuffled pages; the row tables."""
    rng = random.Random(page + dim)
    order = list(range(sum(-(-n // page) for n in lens) + 2))
    cache = ops.Kv8Cache.create(pages=len(order), kv_heads=heads, page_tokens=page, dim=dim)
    rng.shuffle(order)
    width = max(1, max(-(-n // page) for n in lens))
    tables = [[order.pop() for _ in range(-(-n // page))] for n in lens]
    for side in (cache.k_codes, cache.v_codes):
        side.copy_(torch.randint(-127, 128, side.shape, generator=g, device="cuda"))
    for side in (cache.k_scale, cache.v_scale):
        side.copy_((0.5 + torch.rand(side.shape, generator=g, device="cuda")) * 3.0 / 127)
    return cache, ints([t + [-1] * (width - len(t)) for t in tables])


def check(ops, cache, tables, q, lens, cu, *, max_new, scale=None, window=0, softcap=0.0):
    """Every output against 64 bits within the bound at the top of this file; returns (out, lse)."""
    dim, page = cache.dim, cache.page_tokens
    out, lse = ops.kv8_attention(q, cache, tables, ints(lens), ints(cu), max_new=max_new, scale=scale, window=window,
                                 softcap=softcap, return_lse=True)
    scale = dim ** -0.5 if scale is None else scale
    box = 64 if page % 64 == 0 else 32 if page % 32 == 0 else 16
    kvh, group = cache.kv_heads, q.shape[1] // cache.kv_heads
    for r, n in enumerate(lens):
        a, b = cu[r], cu[r + 1]
        held = tables[r, : -(-n // page)].long()

        def rows(x):
            return x[held].double().transpose(0, 1).reshape(kvh, -1, dim)[:, :n]

        def each(x):
            return x[held].double().t().repeat_interleave(page, 1)[:, :n]
        kc, vc, ks, vs = rows(cache.k_codes), rows(cache.v_codes), each(cache.k_scale), each(cache.v_scale)
        low = max(0, n - (b - a) + 1 - window) // box * box if window else 0
        for i in range(a, b):
            pos = n - (b - a) + i - a
            first = max(0, pos - window + 1) if window else 0
            if pos < first:
                assert not out[i].any() and (lse[i] == -math.inf).all()
                continue
            see = slice(first, pos + 1)
            k, v, c = kc[:, see] * ks[:, see, None], vc[:, see] * vs[:, see, None], vc[:, see].abs()
            qi = q[i].double().view(kvh, group, dim)
            x = scale * torch.einsum("hgd,hkd->hgk", qi, k)
            dx = 2.0 ** -30 * abs(scale) * qi.abs().amax(2)[..., None] * k.abs().sum(2)[:, None] + 2.0 ** -21 * (
                abs(scale) * torch.einsum("hgd,hkd->hgk", qi.abs(), k.abs()) + 1)
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            dx = (dx + (2.0 ** -19 + 2.0 ** -21 if softcap else 2.0 ** -21) * x.abs()).amax(2)
            want = torch.logsumexp(x, 2)
            p = torch.exp(x - want[..., None])
            ref = torch.einsum("hgk,hkd->hgd", p, v)
            spread = torch.einsum("hgk,hkd->hgd", p, v.abs())
            steps = torch.zeros_like(ref)
            tile = (torch.arange(first, pos + 1, device="cuda") - low) // 128
            for t in tile.unique().tolist():
                at = tile == t
                top = (p[..., at] * vs[:, None, see][..., at].abs()).amax(2)
                steps += top[..., None] * c[:, at].sum(1)[:, None] * (0.5 / (63 * 2 ** 16))
            bound = HALF_ULP[q.dtype] * ref.abs() + (2 * dx[..., None] + 2.0 ** -20) * spread + 1.01 * steps + SMALLEST[q.dtype]
            far = ((out[i].double().view(ref.shape) - ref).abs() / bound).max().item()
            assert far <= 1.0, (r, i, far)
            assert ((lse[i].double().view(want.shape) - want).abs() <= dx + 2.0 ** -20 * (1 + want.abs())).all()
    assert cache.status() == 0
    return out, lse


# ------------------------------------------------------------------ attention: V scales far apart
def split_scores(cache, tables, light):
    """K codes such that q = 1 scores the keys of the `light` table columns 60 binary orders below the others."""
    dim, page = cache.dim, cache.page_tokens
    cache.k_codes.fill_(40)
    cache.k_codes[tables[0, light].long()] = -40
    cache.k_codes[:, :, :, 0] = torch.randint(-127, 128, cache.k_codes.shape[:3], device="cuda", generator=gen(1))
    cache.k_scale.fill_(1 / 40)
    return 60 * math.log(2) / (2 * (dim - 1))  # the score's scale


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("ratio", [1e2, 1e4, 1e5, 1e8, 2.0 ** 24, 2.0 ** 60])
@pytest.mark.parametrize("dim,heads,page,first_light", [(64, 1, 64, True), (128, 8, 32, False), (256, 16, 16, True), (64, 2, 48, False),
                                                        (128, 16, 128, True)])
def test_small_v_scales_with_all_the_weight(ops, dtype, ratio, dim, heads, page, first_light):
    g = gen(7)
    pages = max(2, 128 // page)
    n = pages * page
    cache, tables = make_cache(ops, g, [n], page, 1, dim)
    half = pages // 2
    light = list(range(half)) if first_light else list(range(half, pages))
    scale = split_scores(cache, tables, light)
    cache.v_scale[tables[0, light].long()] *= ratio
    if dtype is F16:
        cache.v_scale /= max(1.0, ratio / 1e4)  # (the large values stay inside the type)
    q = torch.ones(1, heads, dim, device="cuda").to(dtype)
    q[0, heads // 2:] *= -1.0  # these see the large scales
    check(ops, cache, tables, q, [n], [0, 1], max_new=1, scale=scale)


@pytest.mark.parametrize("page,heads", [(16, 1), (16, 8), (32, 4), (64, 8), (128, 2)])
def test_a_token_does_not_depend_on_the_scale_of_a_page_that_it_does_not_see(ops, page, heads):
    g = gen(page)
    n = page + 1  # the first of two tokens ends a page, the second begins one
    cache, tables = make_cache(ops, g, [n, n], page, 1, 128)
    q = torch.randn(4, heads, 128, generator=g, device="cuda").to(BF16)
    plain, _ = check(ops, cache, tables, q, [n, n], [0, 2, 4], max_new=2)
    for large in (1e3, 1e6, 1e25):  # (up to 2^100 times the others)
        cache.v_scale[tables[0, 1]] = large
        out, _ = check(ops, cache, tables, q, [n, n], [0, 2, 4], max_new=2)
        assert torch.equal(out[0], plain[0]) and torch.equal(out[2:], plain[2:])
    # a scale that is no number: as a page that was never written holds it
    cache.v_scale[tables[0, 1]] = math.nan
    out = ops.kv8_attention(q, cache, tables, ints([n, n]), ints([0, 2, 4]), max_new=2)
    assert torch.equal(out[0], plain[0]) and torch.equal(out[2:], plain[2:]) and torch.isnan(out[1]).all()


@pytest.mark.parametrize("page", [16, 32, 64])
def test_window_over_pages_of_very_different_scales(ops, page):
    g = gen(page + 1)
    lens, new = [900, 300, 128], [2, 1, 40]
    cache, tables = make_cache(ops, g, lens, page, 2, 64)
    exps = torch.randint(-12, 13, cache.v_scale.shape, generator=g, device="cuda").float()
    cache.v_scale *= torch.exp2(exps)
    q = torch.randn(43, 8, 64, generator=g, device="cuda").to(F16) * 3.0
    for window in (0, 17, 100):
        check(ops, cache, tables, q, lens, [0, 2, 3, 43], max_new=40, window=window)
        check(ops, cache, tables, q[:, :2], lens, [0, 2, 3, 43], max_new=2, window=window)


def test_zero_scales_among_others(ops):
    g = gen(3)
    cache, tables = make_cache(ops, g, [256], 32, 1, 128)
    q = torch.randn(1, 8, 128, generator=g, device="cuda").to(F16)
    cache.v_scale[tables[0, ::2].long()] = 0.0
    check(ops, cache, tables, q, [256], [0, 1], max_new=1)
    cache.v_scale[tables[0, 1::2].long()] = 1e-38
    check(ops, cache, tables, q, [256], [0, 1], max_new=1)
    cache.v_scale.zero_()
    out, _ = check(ops, cache, tables, q, [256], [0, 1], max_new=1)
    assert not out.any()


# ------------------------------------------------------------------ attention: q far apart in its row
@pytest.mark.parametrize("ratio", [2.0 ** 10, 2.0 ** 14, 2.0 ** 18, 2.0 ** 21])
@pytest.mark.parametrize("dim,heads,page", [(64, 8, 64), (128, 16, 32), (256, 16, 16)])
def test_a_channel_that_is_large_in_q_and_zero_in_the_keys(ops, ratio, dim, heads, page):
    g = gen(5)
    cache, tables = make_cache(ops, g, [260], page, 1, dim)
    cache.k_codes[..., 7] = 0
    q = torch.randn(2, heads, dim, generator=g, device="cuda").clamp(-3, 3)
    q[:, ::2, 7] = ratio
    q[:, 1::2, 7] = -ratio
    out, _ = check(ops, cache, tables, q.to(BF16), [260], [0, 2], max_new=2)
    q[..., 7] = 0.0
    plain, _ = check(ops, cache, tables, q.to(BF16), [260], [0, 2], max_new=2)
    if ratio <= 2.0 ** 18:  # q's steps (ratio * 2^-29) are far below its elements' own: the same scores, but for single roundings
        assert (out.double() - plain.double()).norm() <= 2.0 ** -9 * plain.double().norm()


# ------------------------------------------------------------------ attention: soft caps of any size
@pytest.mark.parametrize("softcap", [1e-3, 0.5, 7.0, 1e3, 1e4, 1e6, 1e9, 1e20, 3e38])
@pytest.mark.parametrize("dim,heads,page", [(64, 4, 32), (256, 16, 16)])
def test_softcap_of_any_size(ops, softcap, dim, heads, page):
    g = gen(9)
    cache, tables = make_cache(ops, g, [300], page, 1, dim)
    q = torch.randn(1, heads, dim, generator=g, device="cuda").to(F16)
    q *= torch.logspace(-3, 1, heads, device="cuda").to(F16)[:, None]  # scores small and large beside the smaller caps
    check(ops, cache, tables, q, [300], [0, 1], max_new=1, softcap=softcap)


def test_softcaps_that_are_no_cap_are_refused(ops):
    cache, tables = make_cache(ops, gen(1), [16], 16, 1, 64)
    q = torch.zeros(1, 1, 64, device="cuda").to(BF16)
    for softcap in (-1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            ops.kv8_attention(q, cache, tables, ints([16]), ints([0, 1]), max_new=1, softcap=softcap)


# ------------------------------------------------------------------ plans that no longer fit
def state(d):
    return [t.tolist() for t in (d.tables, d.lengths, d.used)]


def test_a_plan_that_no_longer_fits_is_not_committed(ops, pkg):
    from gemma4_omni_b200 import _lib
    stale = _lib.DEV_STALE_COMMIT

    def directory():
        d = ops.PageDirectory.create(sessions=4, max_pages=3, pages=8, page_tokens=16)
        d.commit(d.plan(ints([0, 1]), ints([5, 20]), max_tokens=25))
        assert d.lengths.tolist() == [5, 20, 0, 0]
        return d

    def late(d, plan):
        """The plan is refused and changes nothing."""
        before = state(d)
        d.commit(plan)
        assert plan.status() == stale and state(d) == before
        d.commit(plan)
        assert plan.status() == stale and state(d) == before

    d = directory()  # two plans give the same free pages to different sessions
    a, b = (d.plan(ints([s, 3 - s]), ints([17, 0]), max_tokens=17) for s in (2, 3))
    d.commit(a)
    assert a.status() == 0 and d.lengths.tolist() == [5, 20, 17, 0]
    late(d, b)
    d = directory()  # two plans for the same tokens of a session, inside a page
    a, b = (d.plan(ints([0]), ints([1]), max_tokens=1) for _ in range(2))
    d.commit(a)
    late(d, b)
    late(d, a)  # and one that was committed before
    d = directory()  # a release in between
    a = d.plan(ints([1]), ints([2]), max_tokens=2)
    d.release(ints([1]))
    late(d, a)
    d = directory()  # a release, and the same number of tokens in other pages
    a = d.plan(ints([1]), ints([2]), max_tokens=2)
    d.release(ints([0, 1]))
    d.commit(d.plan(ints([1]), ints([20]), max_tokens=20))
    late(d, a)
    d = directory()  # one row of many
    a = d.plan(ints([2, 0, 3]), ints([40, 3, 1]), max_tokens=44)
    d.commit(d.plan(ints([0]), ints([1]), max_tokens=1))
    late(d, a)
    d = directory()  # other sessions' tokens within their pages do not matter, nor do rows without tokens
    a = d.plan(ints([2, 1]), ints([3, 0]), max_tokens=3)
    d.commit(d.plan(ints([0]), ints([1]), max_tokens=1))
    d.commit(a)
    assert a.status() == 0 and d.lengths.tolist() == [6, 20, 3, 0]


def test_a_late_commit_through_the_entry_without_token_counts(ops, pkg):
    from gemma4_omni_b200 import _lib
    d = ops.PageDirectory.create(sessions=2, max_pages=3, pages=8, page_tokens=16)
    a, b = (d.plan(ints([s]), ints([17]), max_tokens=17) for s in (0, 1))
    for plan, want, lengths in ((a, 0, [17, 0]), (b, _lib.DEV_STALE_COMMIT, [17, 0])):
        _lib.check("lb_commit_pages", _lib.load().lb_commit_pages(
            1, plan.sessions.data_ptr(), 2, 3, 8, 16, plan.row_tables.data_ptr(), plan.kv_len.data_ptr(), plan.status_word.data_ptr(),
            d.tables.data_ptr(), d.lengths.data_ptr(), d.used.data_ptr(), torch.cuda.current_stream().cuda_stream))
        assert plan.status() == want and d.lengths.tolist() == lengths


def test_a_plan_keeps_its_sessions_when_the_callers_buffer_is_filled_anew(ops):
    d = ops.PageDirectory.create(sessions=4, max_pages=3, pages=8, page_tokens=16)
    ids = ints([2, 0])
    plan = d.plan(ids, ints([5, 17]), max_tokens=22)
    ids.copy_(ints([1, 3]))
    assert plan.sessions.tolist() == [2, 0]
    d.commit(plan)
    assert plan.status() == 0 and d.lengths.tolist() == [17, 0, 5, 0]
    assert d.tables.tolist() == [[1, 2, -1], [-1] * 3, [0, -1, -1], [-1] * 3]


# ------------------------------------------------------------------ tensors that are exchanged
def test_tensors_that_do_not_fit_are_refused_when_they_are_set(ops):
    d = ops.PageDirectory.create(sessions=4, max_pages=3, pages=40, page_tokens=16)
    cache = ops.Kv8Cache.create(pages=4, kv_heads=2, page_tokens=16, dim=64)
    weight = ops.Int4Weight.quantize(torch.randn(8, 256, generator=gen(1), device="cuda"))
    for owner, names in ((d, ("tables", "lengths", "used")), (weight, ("codes", "scales")),
                         (cache, ("k_codes", "v_codes", "k_scale", "v_scale", "status_word"))):
        for name in names:
            held = getattr(owner, name)
            twice = torch.cat([held, held], -1)
            # (a single element has no stride)
            for bad in (held[:-1].clone(), twice[..., ::2] if held.numel() > 1 else twice, held.to(torch.int64), held.cpu(), twice, None,
                        torch.zeros(held.numel() + 1, dtype=held.dtype, device="cuda")[1:].view(held.shape) if name.endswith("codes") else held[:0]):
                with pytest.raises(ValueError):
                    setattr(owner, name, bad)
                assert getattr(owner, name) is held
            other = held.clone()
            setattr(owner, name, other)
            assert getattr(owner, name) is other


def test_commit_refuses_plans_whose_tensors_do_not_fit(ops):
    d = ops.PageDirectory.create(sessions=4, max_pages=3, pages=8, page_tokens=16)
    for name in ("sessions", "row_tables", "kv_len", "cu_tokens", "status_word"):
        plan = d.plan(ints([0, 1]), ints([5, 20]), max_tokens=25)
        held = getattr(plan, name)
        for bad in (held[:-1].clone(), held.long(), held.cpu()):
            setattr(plan, name, bad)
            with pytest.raises(ValueError):
                d.commit(plan)
    assert d.lengths.tolist() == [0] * 4


# ------------------------------------------------------------------ append: a page met twice
@pytest.mark.parametrize("heads,pad", [(1, 0), (8, 300), (1, 4000)])
@pytest.mark.parametrize("slots,good", [
    ([16, -1, 17, 32, 33], [0, 3, 4]),              # a skipped token inside a page
    ([16, 17, 19, 20, 5], [0, 1, 4]),               # a gap
    ([18, 17, 33, 34], [0, 2, 3]),                  # a step back
    ([20, 20, 40], [0, 2]),                         # a slot twice
    ([15, 16, 17, -7, 31, -1, -2, 32], [0, 1, 2, 7]),  # pages that end and begin beside them
    ([-1] * 70 + [16] + [-1] * 70 + [17, 48], [70, 142]),  # skipped tokens past the window that a CTA looks at
])
def test_the_tokens_of_a_page_after_a_gap_are_refused(ops, pkg, slots, good, heads, pad):
    from gemma4_omni_b200 import _lib
    slots = [-1] * pad + slots
    good = [pad + i for i in good]
    cache = ops.Kv8Cache.create(pages=4, kv_heads=heads, page_tokens=16, dim=64)
    want = ops.Kv8Cache.create(pages=4, kv_heads=heads, page_tokens=16, dim=64)
    for c in (cache, want):  # what the pages held
        for t in (c.k_codes, c.v_codes):
            t.copy_(torch.randint(-127, 128, t.shape, generator=gen(2), device="cuda"))
        c.k_scale.fill_(0.001)
        c.v_scale.fill_(0.01)
    x = torch.randn(len(slots), heads, 64, generator=gen(1), device="cuda")
    cache.append(x, -x, torch.tensor(slots, device="cuda"))
    kept = torch.full((len(slots),), -1, device="cuda")
    kept[good] = torch.tensor(slots, device="cuda")[good]
    want.append(x, -x, kept)
    assert cache.status() == (_lib.DEV_SPLIT_PAGE if len(good) < sum(s >= 0 for s in slots) else 0)
    if want.status() == 0:
        for name in ("k_codes", "v_codes", "k_scale", "v_scale"):
            assert torch.equal(getattr(cache, name), getattr(want, name)), name


# ------------------------------------------------------------------ norm: codes are those of the quotient
def quotient_codes(w, scale, out):
    """round(w / scale) by IEEE division in 32 bits, to nearest even."""
    q = torch.div(w, scale.expand_as(w))
    return q.round().clamp(-127, 127).to(I8) if out is I8 else q.clamp(-448, 448).to(E4M3)


@pytest.mark.parametrize("out", [E4M3, I8])
@pytest.mark.parametrize("dim,group,offset", [(4096, 0, 0), (2048, 128, 0), (256, 8, 0), (1024, 0, 1), (2048, 64, 3)])
@pytest.mark.parametrize("rows", [1, 1200])
def test_codes_are_the_rounded_quotient(ops, out, dim, group, offset, rows):
    """Rows of ones have the norm 1, so that y is the weight itself, exactly; many quotients lie halfway."""
    g = gen(dim + group)
    top = 448 if out is E4M3 else 127
    x = torch.ones(rows, dim + offset, device="cuda")[:, offset:]
    whole = torch.randint(-top, top + 1, (dim,), generator=g, device="cuda").float()
    for k, w in enumerate((whole + 0.5 * torch.randint(0, 2, (dim,), generator=g, device="cuda"), whole * 3.0, whole * 2.0 ** -100,
                           torch.randn(dim, generator=g, device="cuda").to(BF16).float(), torch.randn(dim, generator=g, device="cuda") * 1e3,
                           torch.randn(dim, generator=g, device="cuda") * 1e30)):
        if k in (0, 1, 2):
            w[::max(8, group or dim)] = top * (1.0, 6.0, 2.0 ** -100)[k]  # the scale is 1, 6 or 2^-100 in every group
        codes, scales, _ = ops.rms_norm8(x, w, eps=0.0, group=group, dtype=out)
        s = scales.repeat_interleave(group or dim, 1)
        want = quotient_codes(w.expand(rows, dim), s, out)
        assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)), k
        torch.testing.assert_close(scales[0].double(), w.double().abs().view(-1, group or dim).amax(1) / top, rtol=2.0 ** -22, atol=0)


@pytest.mark.parametrize("out", [E4M3, I8])
@pytest.mark.parametrize("offset", [0, 1])
def test_a_group_with_an_infinite_value_has_codes_of_zero(ops, out, offset):
    x = torch.ones(2, 256 + offset, device="cuda")[:, offset:]
    w = torch.ones(256, device="cuda")
    w[3], w[200] = math.inf, -2.0
    codes, scales, _ = ops.rms_norm8(x, w, eps=0.0, group=128, dtype=out)
    assert torch.isinf(scales[:, 0]).all() and not codes[:, :128].view(torch.uint8).any()
    assert torch.equal(codes[:, 128:].view(torch.uint8), quotient_codes(w[128:].expand(2, 128), scales[:, 1:].expand(2, 128), out).view(torch.uint8))


# ------------------------------------------------------------------ attention: rows that see nothing, windows, tokens
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_a_token_that_sees_no_key_gets_zeros_whatever_its_query_holds(ops, page, softcap):
    cache, tables = make_cache(ops, gen(1), [40, 1, 300], page, 1, 64)
    q = torch.full((8, 4, 64), math.nan, device="cuda").to(BF16)
    q[4], q[6] = 1.0, math.inf
    # rows: one without keys, one with more tokens than keys, one whose last token is the only one with numbers
    out, lse = ops.kv8_attention(q, cache, tables, ints([0, 2, 300]), ints([0, 1, 5, 8]), max_new=4, softcap=softcap, return_lse=True)
    assert not out[:3].any() and (lse[:3] == -math.inf).all()
    assert torch.isnan(out[3]).all() and torch.isfinite(out[4]).all() and torch.isnan(out[5:]).all()


@pytest.mark.parametrize("window", [300, 2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5])
@pytest.mark.parametrize("lens,new", [([300, 20], [3, 1]), ([3, 5], [7, 130])])
def test_windows_wider_than_all_keys_hide_none(ops, window, lens, new):
    g = gen(4)
    cache, tables = make_cache(ops, g, [max(n, m) for n, m in zip(lens, new)], 32, 1, 64)
    q = torch.randn(sum(new), 2, 64, generator=g, device="cuda").to(F16)
    kv_len, cu = ints(lens), ints([0, new[0], sum(new)])
    want = ops.kv8_attention(q, cache, tables, kv_len, cu, max_new=max(new), return_lse=True)
    got = ops.kv8_attention(q, cache, tables, kv_len, cu, max_new=max(new), window=window, return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_a_hint_past_32_bits(ops):
    g = gen(4)
    cache, tables = make_cache(ops, g, [50], 32, 1, 64)
    q = torch.randn(20, 1, 64, generator=g, device="cuda").to(F16)
    want = ops.kv8_attention(q, cache, tables, ints([50]), ints([0, 20]), max_new=20)
    for hint in (2 ** 31, 2 ** 32, 2 ** 40):
        assert torch.equal(ops.kv8_attention(q, cache, tables, ints([50]), ints([0, 20]), max_new=hint), want)


@pytest.mark.parametrize("window", [0, 20])
def test_q_may_end_before_the_last_rows_tokens_do(ops, window):
    """A step's first tokens alone: each stays at its own position."""
    g = gen(6)
    cache, tables = make_cache(ops, g, [90, 130], 32, 1, 64)
    q = torch.randn(40, 4, 64, generator=g, device="cuda").to(F16)
    lens, cu = [90, 130], [0, 10, 40]
    whole, _ = check(ops, cache, tables, q, lens, cu, max_new=30, window=window)
    for t in (1, 9, 10, 11, 39):
        part = ops.kv8_attention(q[:t], cache, tables, ints(lens), ints(cu), max_new=30, window=window)
        torch.testing.assert_close(part, whole[:t], rtol=2.0 ** -10, atol=1e-5)


# ------------------------------------------------------------------ shapes and strides of the wrappers
def test_single_rows_and_columns_of_any_stride(ops):
    """What torch calls a row's stride does not matter where there is one row, nor a column's where there is one."""
    g = gen(3)
    w = ops.Int4Weight.quantize(torch.randn(8, 128, generator=g, device="cuda"))
    col = torch.randn(128, 1, generator=g, device="cuda").to(BF16)
    x, ones = col.t(), torch.ones(128, device="cuda")  # [1, 128] with strides (1, 1)
    assert x.stride() == (1, 1)
    plain = x.clone(memory_format=torch.contiguous_format).view(1, 128)
    for a, b in zip(ops.rms_norm8(x, ones, residual=x), ops.rms_norm8(plain.reshape(1, 128), ones, residual=plain)):
        assert torch.equal(a.view(-1).float(), b.view(-1).float())
    out = torch.zeros(8, 1, device="cuda").t()
    ops.w4_matvec(x, w, out=out)
    assert torch.equal(out, ops.w4_matvec(torch.empty(1, 128, device="cuda", dtype=BF16).copy_(x), w, out_dtype=F32))
    narrow = torch.randn(5, 3, generator=g, device="cuda")[:, 1:2]  # [5, 1] with strides (3, 1)
    for a, b in zip(ops.rms_norm8(narrow, ones[:1]), ops.rms_norm8(narrow.contiguous(), ones[:1])):
        assert torch.equal(a.float(), b.float())
    turned = torch.randn(1, 5, generator=g, device="cuda").t()[:, :1].as_strided((5, 1), (1, 7))
    for a, b in zip(ops.rms_norm8(turned, ones[:1]), ops.rms_norm8(turned.clone(memory_format=torch.contiguous_format), ones[:1])):
        assert torch.equal(a.float(), b.float())


def test_rows_that_overlap_are_refused(ops):
    w = ops.Int4Weight.quantize(torch.zeros(8, 128, device="cuda"))
    ones = torch.ones(128, device="cuda")
    one = torch.zeros(1, 128, device="cuda")
    for f in (lambda: ops.rms_norm8(one.expand(3, 128), ones),
              lambda: ops.rms_norm8(torch.zeros(3, 128, device="cuda"), ones, residual=one.expand(3, 128)),
              lambda: ops.w4_matvec(one.to(BF16).expand(3, 128), w),
              lambda: ops.w4_matvec(torch.zeros(3, 128, device="cuda").to(BF16), w, out=torch.zeros(1, 8, device="cuda").expand(3, 8))):
        with pytest.raises(ValueError):
            f()


def test_a_step_of_the_block_without_tokens(pkg):
    """A tick in which no session has anything new."""
    from gemma4_omni_b200.decode_ops import PageDirectory
    from gemma4_omni_b200.decoder_block import DecoderBlock, DecoderConfig
    block = DecoderBlock.synthetic(DecoderConfig(hidden=256, heads=4, kv_heads=2, head_dim=64, ffn=512), seed=1)
    pages = PageDirectory.create(sessions=2, max_pages=2, pages=4, page_tokens=16)
    cache = block.new_cache(4, 16)
    plan = pages.plan(ints([0, 1]), ints([0, 0]), max_tokens=1)
    y = block.step(torch.zeros(0, 256, dtype=BF16, device="cuda"), plan, cache, max_new=1)
    pages.commit(plan)
    assert y.shape == (0, 256) and plan.status() == 0 and pages.lengths.tolist() == [0, 0]


def test_keys_past_a_rows_table_are_said_to_be_missing(ops, pkg):
    from gemma4_omni_b200 import _lib
    g = gen(8)
    cache, tables = make_cache(ops, g, [64, 10], 16, 1, 64)
    q = torch.randn(2, 2, 64, generator=g, device="cuda").to(F16)
    ops.kv8_attention(q, cache, tables, ints([64, 10]), ints([0, 1, 2]), max_new=1)
    assert cache.status() == 0
    ops.kv8_attention(q, cache, tables, ints([65, 10]), ints([0, 1, 2]), max_new=1)
    assert cache.status() == _lib.DEV_BAD_PAGE
    cache.status_word.zero_()
    ops.kv8_attention(q, cache, tables, ints([65, 10]), ints([0, 0, 1]), max_new=1)  # a row without tokens reads nothing
    assert cache.status() == 0


# ------------------------------------------------------------------ bounds that a lost digit or column would pass
SHAPES = [  # dim, kv heads, group, page, lens, new, window, softcap
    (64, 1, 1, 16, [1], [1], 0, 0.0),
    (128, 1, 1, 64, [0, 1, 2, 15, 16, 17], [1, 1, 2, 1, 0, 1], 0, 0.0),
    (256, 1, 8, 64, [700, 64, 63, 65, 2, 1], [2, 2, 1, 2, 2, 1], 0, 0.0),
    (128, 8, 4, 32, [1000, 33, 257], [1, 1, 1], 0, 0.0),
    (64, 2, 3, 48, [500, 47, 49, 97], [1, 2, 3, 1], 0, 50.0),
    (128, 2, 16, 16, [300, 20], [3, 2], 17, 0.0),
    (256, 2, 1, 128, [3000, 5], [1, 1], 1000, 30.0),
    (64, 4, 2, 256, [515, 260, 100], [130, 1, 100], 0, 0.0),
    (128, 1, 2, 16, [3, 0, 5], [7, 4, 9], 0, 0.0),
    (128, 1, 8, 64, [9000], [1], 0, 0.0),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_is_as_close_as_its_digits_say(ops, dtype, shape):
    dim, kvh, group, page, lens, new, window, softcap = SHAPES[shape]
    g = gen(shape)
    cache, tables = make_cache(ops, g, [max(n, 1) for n in lens], page, kvh, dim)
    q = torch.randn(sum(new), kvh * group, dim, generator=g, device="cuda").to(dtype)
    check(ops, cache, tables, q, lens, [sum(new[:i]) for i in range(len(new) + 1)], max_new=max(new), window=window, softcap=softcap)


@pytest.mark.parametrize("heads,page", [(1, 16), (8, 64), (16, 32)])
def test_values_that_cancel_show_the_digits_of_p(ops, heads, page):
    """Values of +-127 by turns: the outputs are small beside sum p|v|, so that p's low digits stand above their rounding."""
    g = gen(heads)
    cache, tables = make_cache(ops, g, [4096], page, 1, 64)
    cache.v_codes[:, :, ::2] = 127
    cache.v_codes[:, :, 1::2] = -127
    cache.v_scale.fill_(1 / 127)
    q = 0.1 * torch.randn(1, heads, 64, generator=g, device="cuda").to(F16)
    check(ops, cache, tables, q, [4096], [0, 1], max_new=1)


@pytest.mark.parametrize("page", [16, 64])
def test_two_keys_that_cancel_show_the_last_digit_of_p(ops, page):
    """A weight of about 1 on a value of 1 against one of about 1 / 127 on -127: p without its last digit would be off by up
    to 2^-15 * 127, a hundred times the bound."""
    cache, tables = make_cache(ops, gen(1), [2], page, 1, 64)
    cache.k_codes.zero_()
    at = int(tables[0, 0])
    cache.k_codes[at, 0, 1, 0] = 100
    cache.k_scale.fill_(0.01)
    cache.v_codes[at, 0, 0], cache.v_codes[at, 0, 1] = 1, -127
    cache.v_scale.fill_(1 / 127)
    q = torch.zeros(1, 16, 64, device="cuda")
    q[0, :, 0] = -38.75 + torch.arange(16, device="cuda") / 32.0
    check(ops, cache, tables, q.to(F16), [2], [0, 1], max_new=1)


@pytest.mark.parametrize("kind", [BF16, F16, E4M3, I8])
@pytest.mark.parametrize("out,k,group", [(33, 96, 32), (70, 1536, 128), (257, 320, 64), (32, 6144, 128), (5000, 256, 64), (40, 8192, 32)])
def test_w4_every_column_counts_with_its_own_weight(ops, kind, out, k, group):
    """Rows with a single one in them: the products are the weights, exactly."""
    g = gen(out + k)
    codes = torch.randint(0, 256, (out, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.01 * (0.1 + torch.rand(out, k // group, generator=g, device="cuda"))).to(F16)
    weight = ops.Int4Weight(codes, scales)
    want = weight.dequantize()
    n = min(k, 512)
    at = torch.randperm(k, generator=g, device="cuda")[:n] if k > 512 else torch.arange(k, device="cuda")
    x = torch.zeros(n, k, device="cuda")
    x[torch.arange(n, device="cuda"), at] = 1.0
    xs = torch.ones(n, 1, device="cuda") if kind in (E4M3, I8) else None
    for rows in (n, 16, 3):
        y = ops.w4_matvec(x[:rows].to(kind), weight, x_scale=None if xs is None else xs[:rows], out_dtype=F32)
        assert torch.equal(y, want[:, at[:rows]].t())


@pytest.mark.parametrize("kind", [BF16, F16, I8])
@pytest.mark.parametrize("rows,out,k,group", [(1, 2048, 1536, 128), (2, 100, 512, 64), (9, 33, 2048, 32), (16, 4097, 256, 64), (37, 70, 8192, 128),
                                              (1, 515, 16384, 128), (16, 160, 6144, 128)])
def test_w4_sums_are_within_their_roundings(ops, kind, rows, out, k, group):
    """Products are exact; each of a group's k / 16 additions on the tensor cores is good to 2^-21 of the sum of absolute
    values so far, the groups' sums are added in 32 bits.  One column left out would be 1 / k of the sum."""
    g = gen(rows + k)
    codes = torch.randint(0, 256, (out, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.01 * (0.1 + torch.rand(out, k // group, generator=g, device="cuda"))).to(F16)
    weight = ops.Int4Weight(codes, scales)
    x, xs = torch.randn(rows, k, generator=g, device="cuda"), None
    if kind is I8:
        x, xs, _ = ops.rms_norm8(x, torch.ones(k, device="cuda"), dtype=I8)
    else:
        x = x.to(kind)
    y = ops.w4_matvec(x, weight, x_scale=xs, out_dtype=F32)
    ref, spread = decode_ref.w4_product(x, xs, codes, scales)
    bound = ((group // 16 + 2) * 2.0 ** -21 + (k // group + 18) * 2.0 ** -24) * spread + 1e-30
    assert ((y.double() - ref).abs() <= bound).all()
