"""Norms of queries and keys with their rotation, against the definition in 64 bits.

Bound, from the arithmetic (u = 2^-24): the sum of dim squares, its mean, root and the two products are good to (dim / 8 + 16) u
relative (a lane sums 8 values in order, lanes add up in a tree), sines and cosines to 3 u absolute; so a rotated value
is off by at most (dim / 8 + 24) u (|a| + |b|) and half a step of its type."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import decode_ref

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops(pkg):
    from gemma4_omni_b200 import decode_ops
    return decode_ops


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def check(y, x, weight, positions, frequencies, *, rotary, pairs, eps=1e-6, norm=True):
    ref = decode_ref.head_norm_rotary(x, weight, positions, frequencies, rotary=rotary, pairs=pairs, eps=eps, norm=norm)
    plain = decode_ref.head_norm_rotary(x, weight, torch.zeros_like(positions), frequencies, rotary=rotary, pairs=pairs, eps=eps,
                                        norm=norm).abs()
    size = plain.clone()  # |a| + |b| of a value's pair
    if pairs == "halves":
        size[..., :rotary] += plain[..., :rotary].roll(rotary // 2, -1)
    else:
        size[..., :rotary] += plain[..., :rotary].unflatten(-1, (-1, 2)).flip(-1).flatten(-2)
    tiny = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    bound = torch.finfo(y.dtype).eps / 2 * ref.abs() + (x.shape[2] / 8 + 24) * 2.0 ** -24 * size + tiny
    assert ((y.double() - ref).abs() <= bound).all()


def frequencies(rotary, base):
    return [base ** (-2.0 * i / rotary) for i in range(rotary // 2)]


@pytest.mark.parametrize("tokens,heads,kv,dim,rotary,pairs,dtype,wide,far", [
    (1, 1, 1, 64, 64, "halves", BF16, True, 5), (2, 8, 1, 256, 256, "halves", BF16, True, 20000),
    (5, 5, 3, 128, 128, "halves", F16, False, 1 << 30), (33, 32, 8, 128, 64, "halves", BF16, False, 100000),
    (700, 6, 2, 64, 16, "neighbours", F32, True, 1 << 20), (3, 3, 1, 96, 48, "halves", F32, True, 4096),
    (40, 7, 5, 256, 256, "neighbours", F16, True, 99), (9, 2, 1, 512, 512, "halves", BF16, True, 5000),
    (4, 3, 2, 10, 6, "halves", F32, True, 77), (4, 3, 2, 66, 66, "neighbours", BF16, True, 77), (3, 1, 1, 2, 2, "halves", F16, True, 9),
    (2500, 4, 4, 64, 64, "halves", BF16, True, 1 << 31)])
def test_follows_the_definition(ops, tokens, heads, kv, dim, rotary, pairs, dtype, wide, far):
    g = gen(tokens)
    both = (torch.randn(tokens, heads + 2 * kv, dim, generator=g, device="cuda") * 3).to(dtype)
    q, k, v = both.split((heads, kv, kv), 1)
    w = [(1 + 0.3 * torch.randn(dim, generator=g, device="cuda")).to(F32 if wide else dtype) for _ in range(2)]
    at = torch.randint(0, far, (tokens,), generator=g, device="cuda", dtype=torch.int64)
    at = at if far > 1 << 30 else at.to(torch.int32)
    r = ops.Rotary.create(dim, rotary_dim=rotary, base=50000.0, pairs=pairs)
    before = both.clone()
    yq, yk = ops.head_norm_rotary(q, k, at, r, q_weight=w[0], k_weight=w[1])
    assert torch.equal(both, before)
    check(yq, q, w[0], at, frequencies(rotary, 50000.0), rotary=rotary, pairs=pairs)
    check(yk, k, w[1], at, frequencies(rotary, 50000.0), rotary=rotary, pairs=pairs)


@pytest.mark.parametrize("dim", [64, 128, 256, 34])
def test_in_place_and_other_layouts(ops, dim):
    """Outputs over their inputs, heads before tokens, rows off their alignment: the same bits."""
    g = gen(dim)
    q = torch.randn(19, 6, dim, generator=g, device="cuda").to(BF16)
    k = torch.randn(19, 2, dim, generator=g, device="cuda").to(BF16)
    at = torch.arange(19, device="cuda", dtype=torch.int32) * 1000
    r = ops.Rotary.create(dim, base=1e6)
    yq, yk = ops.head_norm_rotary(q, k, at, r)
    both = torch.cat([q, k], 1)
    a, b = both.split((6, 2), 1)
    ops.head_norm_rotary(a, b, at, r, q_out=a, k_out=b)
    assert torch.equal(a, yq) and torch.equal(b, yk)
    t = q.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.zeros(6, 19, dim, dtype=BF16, device="cuda").transpose(0, 1)
    assert torch.equal(ops.head_norm_rotary(t, None, at, r, q_out=out)[0], yq) and torch.equal(out, yq)
    room = torch.zeros(19, 6 * dim + 3, dtype=BF16, device="cuda")
    odd = room[:, 1:1 + 6 * dim].unflatten(1, (6, dim))
    odd.copy_(q)
    z, none = ops.head_norm_rotary(odd, None, at, r)
    # (other lanes hold other values, so sums have another order)
    assert none is None and (z.float() - yq.float()).abs().max() <= 2.0 ** -7 * yq.float().abs().max()
    one = q[:, :1].expand(19, 6, dim)  # a broadcast input
    z, _ = ops.head_norm_rotary(one, None, at, r)
    assert torch.equal(z, yq[:, :1].expand(19, 6, dim))


def test_values_of_the_ends(ops):
    """Rows of zeros, of the largest and smallest values, with NaN; positions negative and beyond 32 bits; without the norm."""
    r = ops.Rotary.create(64, base=10000.0)
    x = torch.zeros(6, 1, 64, device="cuda")
    x[1], x[2], x[3, 0, 5], x[4] = 1e18, 1e-30, math.nan, torch.randn(64, device="cuda")
    x[5] = x[4]
    at = torch.tensor([7, 0, 3, 4, -(1 << 40), 1 << 40], device="cuda")
    y, _ = ops.head_norm_rotary(x, None, at, r)
    assert (y[0] == 0).all() and torch.isnan(y[3]).all() and torch.isfinite(y[[0, 1, 2, 4, 5]]).all()
    assert (y[1] - 1).abs().max() < 1e-5
    y, _ = ops.head_norm_rotary(x, None, at, r, norm=False)
    # exact angles of far positions, by whole numbers
    exact = [(int(p) * (t % 2 ** 64) % 2 ** 64) / 2 ** 64 * 2 * math.pi for p in (-(1 << 40), 1 << 40) for t in r.turns.tolist()]
    angle = torch.tensor(exact, dtype=torch.float64, device="cuda").view(2, 32)
    a, b = x[4:, 0, :32].double(), x[4:, 0, 32:].double()
    ref = torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], 1)
    assert (y[4:, 0].double() - ref).abs().max() <= 8 * 2.0 ** -24 * x[4].abs().max() * 2
    assert torch.equal(y[1], ops.head_norm_rotary(x[1:2], None, at[1:2], r, norm=False)[0][0])


def test_far_positions_against_the_frequencies(ops):
    """The angle's own bound: 2^-65 turns times the position for the frequency's rounding, 2^-32 turns for the bits that are dropped; beside it
    six roundings of 2^-24 (sines 3, the products and sums)."""
    import decimal
    pi = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803")
    at = [12345, (1 << 31) - 1, -(1 << 31), (1 << 40) + 3, -(1 << 44) - 7, (1 << 50) + 11]
    with decimal.localcontext() as c:
        c.prec = 80
        angles = [[float((p * decimal.Decimal(10000) ** (decimal.Decimal(-2 * i) / 64)) % (2 * pi)) for i in range(32)] for p in at]
    angle = torch.tensor(angles, dtype=torch.float64, device="cuda")
    x = torch.randn(len(at), 1, 64, generator=gen(8), device="cuda")
    y, _ = ops.head_norm_rotary(x, None, torch.tensor(at, device="cuda"), ops.Rotary.create(64), norm=False)
    a, b = x[:, 0, :32].double(), x[:, 0, 32:].double()
    ref = torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], 1)
    off = 2 * math.pi * (torch.tensor(at, dtype=torch.float64, device="cuda").abs() * 2.0 ** -65 + 2.0 ** -32)[:, None] + 6 * 2.0 ** -24
    size = (a.abs() + b.abs()).repeat(1, 2)
    assert ((y[:, 0].double() - ref).abs() <= off * size).all()


def test_rotation_keeps_scores_of_equal_distances(ops):
    """q at p + d and k at p have the same product for every p: 2 dim products of values good to some 2^-22."""
    g = gen(5)
    q, k = (torch.randn(1, 1, 128, generator=g, device="cuda").expand(50, 1, 128) for _ in range(2))
    at = torch.arange(50, device="cuda") * 123457
    r = ops.Rotary.create(128, base=1e6)
    y, _ = ops.head_norm_rotary(q, None, at + 321, r)
    z, _ = ops.head_norm_rotary(k, None, at, r)
    scores = (y * z).double().sum(2)
    assert (scores - scores[0]).abs().max() <= 128 * 2.0 ** -21


def test_given_frequencies_are_those_of_create(ops):
    a = ops.Rotary.create(64, rotary_dim=32, base=10000.0)
    b = ops.Rotary.from_frequencies(frequencies(32, 10000.0), 64)
    step = (a.turns - b.turns).abs()  # a double's frequency is good to 2^-53 of a radian, a turn has 2^64 steps
    assert int(step.max()) <= 2 ** 10
    c = ops.Rotary.from_frequencies(torch.tensor([0.0, 2 * math.pi * 3, -1.0]), 8)
    assert c.turns[0] == 0 and abs(int(c.turns[1])) < 2 ** 42 and int(c.turns[2]) < 0


def test_graph_streams_and_refusals(ops):
    r = ops.Rotary.create(64)
    q, k = torch.randn(4, 4, 64, device="cuda").to(BF16), torch.randn(4, 2, 64, device="cuda").to(BF16)
    at = torch.arange(4, device="cuda", dtype=torch.int32)
    want = ops.head_norm_rotary(q, k, at, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.head_norm_rotary(q, k, at, r)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.head_norm_rotary(q, k, at, r)
    at.add_(5)
    graph.replay()
    later = ops.head_norm_rotary(q, k, at, r)
    assert torch.equal(out[0], later[0]) and torch.equal(out[1], later[1]) and not torch.equal(out[0], want[0])
    assert ops.head_norm_rotary(q[:0], k[:0], at[:0], r)[0].shape == (0, 4, 64)
    w = torch.ones(64, device="cuda")
    for bad in (lambda: ops.head_norm_rotary(q.double(), None, at, r), lambda: ops.head_norm_rotary(q[..., :32], None, at, r),
                lambda: ops.head_norm_rotary(q, k[:3], at, r), lambda: ops.head_norm_rotary(q, k.half(), at, r),
                lambda: ops.head_norm_rotary(q, k, at[:3], r), lambda: ops.head_norm_rotary(q, k, at.float(), r),
                lambda: ops.head_norm_rotary(q, k, at.cpu(), r), lambda: ops.head_norm_rotary(q, k, at, r, q_weight=w[:32]),
                lambda: ops.head_norm_rotary(q, k, at, r, q_weight=w.half()),
                lambda: ops.head_norm_rotary(q, k, at, r, q_weight=w, k_weight=w.to(BF16)),
                lambda: ops.head_norm_rotary(q, None, at, r, k_weight=w), lambda: ops.head_norm_rotary(q, k, at, r, eps=-1.0),
                lambda: ops.head_norm_rotary(q, k, at, r, q_weight=w, norm=False),
                lambda: ops.head_norm_rotary(q, k, at, r, q_out=q.float()),
                lambda: ops.head_norm_rotary(q, k, at, r, q_out=q[:, :1].expand(4, 4, 64)),
                lambda: ops.head_norm_rotary(q.transpose(1, 2), None, at, r), lambda: ops.Rotary.create(64, rotary_dim=66),
                lambda: ops.Rotary.create(64, pairs="thirds"), lambda: ops.Rotary.create(64, base=-1.0),
                lambda: ops.Rotary.create(2048), lambda: ops.Rotary.from_frequencies([math.inf], 8),
                lambda: setattr(r, "turns", r.turns[:3])):
        with pytest.raises(ValueError):
            bad()


def test_outputs_that_share_memory_are_refused(ops):
    """Parts of one buffer: beside one another they may be inputs and outputs in any way, over one another only an input's own output."""
    r = ops.Rotary.create(64)
    at = torch.arange(5, device="cuda", dtype=torch.int32)
    room = torch.randn(5, 20, 64, device="cuda").to(BF16)
    q, k = room[:, :6], room[:, 6:8]
    want = ops.head_norm_rotary(q, k, at, r)
    before = room.clone()
    for bad in (dict(q_out=room[:, 1:7]), dict(q_out=room[:, 2:8]), dict(k_out=room[:, 5:7]), dict(k_out=room[:, :2]), dict(q_out=room[:, 7:13]),
                dict(q_out=room[:, 8:14], k_out=room[:, 13:15]), dict(q_out=room.view(5, 10, 128)[:, 2:8, :64]),
                dict(q_out=room.view(-1)[32:32 + 5 * 6 * 64].view(5, 6, 64))):
        with pytest.raises(ValueError):
            ops.head_norm_rotary(q, k, at, r, **bad)
    with pytest.raises(ValueError):
        ops.head_norm_rotary(q, q, at, r, q_out=q)
    assert torch.equal(room, before)
    for good in (dict(q_out=room[:, 8:14], k_out=room[:, 14:16]), dict(q_out=room.view(5, 10, 128)[:, 4:, :64], k_out=room[:, 9:12:2]), dict(k_out=k),
                 dict(q_out=q), dict(q_out=q, k_out=k)):
        room.copy_(before)
        got = ops.head_norm_rotary(q, k, at, r, **good)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_outputs_that_share_memory_are_refused(ops):
    """Parts of one buffer: beside one another they may be inputs and outputs in any way, over one another only an input's own output."""
    from gemma4_omni_b200._lib import ListenerLibError
    r = ops.Rotary.create(64)
    at = torch.arange(5, device="cuda", dtype=torch.int32)
    room = torch.randn(5, 20, 64, device="cuda").to(BF16)
    q, k = room[:, :6], room[:, 6:8]
    want = ops.head_norm_rotary(q, k, at, r)
    before = room.clone()
    for bad in (dict(q_out=room[:, 1:7]), dict(q_out=room[:, 2:8]), dict(k_out=room[:, 5:7]), dict(k_out=room[:, :2]), dict(q_out=room[:, 7:13]),
                dict(q_out=room[:, 8:14], k_out=room[:, 13:15]), dict(q_out=room.view(5, 10, 128)[:, 2:8, :64]),
                dict(q_out=room.view(-1)[32:32 + 5 * 6 * 64].view(5, 6, 64))):
        with pytest.raises(ListenerLibError):
            ops.head_norm_rotary(q, k, at, r, **bad)
    with pytest.raises(ListenerLibError):
        ops.head_norm_rotary(q, q, at, r, q_out=q)
    assert torch.equal(room, before)
    for good in (dict(q_out=room[:, 8:14], k_out=room[:, 14:16]), dict(q_out=room.view(5, 10, 128)[:, 4:, :64], k_out=room[:, 9:12:2]), dict(k_out=k),
                 dict(q_out=q), dict(q_out=q, k_out=k)):
        room.copy_(before)
        got = ops.head_norm_rotary(q, k, at, r, **good)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_layouts_in_one_buffer(ops):
    """Inputs and outputs at random places of one buffer, with one step between tokens: refused where any value is shared, right otherwise.
    (Rows of another alignment take another kernel: twice the bound above with |a| + |b| <= 2 sqrt(8), less than 2^-15.)"""
    import random
    from gemma4_omni_b200._lib import ListenerLibError
    rng, r, dim = random.Random(6), ops.Rotary.create(8), 8
    room = torch.randn(4000, device="cuda")
    numbers = torch.arange(4000)
    at = torch.arange(3, device="cuda", dtype=torch.int32)
    done = {True: 0, False: 0}
    for _ in range(400):
        token = rng.choice([40, 64, 100, 300])
        hq, hk = rng.randint(1, 4), rng.randint(1, 2)
        places = []
        for heads in (hq, hk, hq, hk):
            head = rng.choice([8, 8, 12, 16, 24])
            places.append(((3, heads, dim), (token, head, 1), rng.randint(0, 300)))
        if token < max(p[1][1] * (p[0][1] - 1) + dim for p in places):
            continue
        sets = [set(numbers.as_strided(*p).flatten().tolist()) for p in places]
        bad = bool(sets[2] & (sets[0] | sets[1]) or sets[3] & (sets[0] | sets[1] | sets[2]))
        q, k, q_out, k_out = (room.as_strided(*p) for p in places)
        want = ops.head_norm_rotary(q.clone(), k.clone(), at, r)
        if bad:
            with pytest.raises((ValueError, ListenerLibError)):  # (the first for one that begins where its input does, with other strides)
                ops.head_norm_rotary(q, k, at, r, q_out=q_out, k_out=k_out)
        else:
            ops.head_norm_rotary(q, k, at, r, q_out=q_out, k_out=k_out)
            assert (q_out - want[0]).abs().max() <= 2.0 ** -15 and (k_out - want[1]).abs().max() <= 2.0 ** -15
        done[bad] += 1
    assert min(done.values()) > 30
