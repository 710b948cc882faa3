"""The gated product with 4-bit weights against its definition in 64 bits.

Bound, from the arithmetic: a product's k terms are exact and summed in 32 bits, at most k additions and k / 32 steps of a scale,
each off by 2^-23 of the sum of absolute values at most, so e = (k + k / 32 + 4) 2^-23 (the last: the scales of x); the activation is
good to 2^-20 of itself, the product of the two and the store to half a step of the output's type each."""
from __future__ import annotations

import math

import pytest
import torch

from helpers import exact_gated_case, exact_gated_limit
from oracle import decode_ref

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3, I8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8
TOP = {E4M3: 448.0, I8: 127.0}


@pytest.fixture(scope="module")
def ops(pkg):
    from gemma4_omni_b200 import decode_ops
    return decode_ops


def inputs(ops, rows, k, ffn, group, x_type, x_group, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    codes = torch.randint(0, 256, (2 * ffn, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = ((0.5 + torch.rand(2 * ffn, k // group, generator=g, device="cuda")) * (0.25 * k ** -0.5)).to(F16)
    x, xs = torch.randn(rows, k, generator=g, device="cuda"), None
    if x_type in TOP:
        xg = x.view(rows, -1, x_group or k)
        xs = xg.abs().amax(2) / TOP[x_type]
        x = (xg / xs[:, :, None]).view(rows, k).clamp(-TOP[x_type], TOP[x_type])
        x = x.round() if x_type == I8 else x
    return x.to(x_type), xs, ops.Int4Weight(codes, scales)


def check(out, x, xs, weight, activation):
    ref, bound = decode_ref.gated(x, xs, weight.codes, weight.scales, activation=activation)
    t = torch.finfo(out.dtype)
    limit = bound((weight.k + weight.k / 32 + 4) * 2.0 ** -23) + (t.eps / 2 + 2.0 ** -20 + 2.0 ** -23) * ref.abs() + t.smallest_normal * t.eps
    assert ((out.double() - ref).abs() <= limit).all()
    assert weight.status() == 0


@pytest.mark.parametrize("x_type,x_group", [(BF16, 0), (F16, 0), (E4M3, 0), (I8, 0), (E4M3, 128), (I8, 256)])
@pytest.mark.parametrize("rows,k,ffn,group", [
    (1, 256, 128, 128), (2, 1536, 6144, 128), (3, 512, 100, 64), (32, 768, 129, 32), (33, 256, 300, 128), (64, 1024, 640, 64),
    (65, 512, 130, 32), (129, 1536, 257, 128), (300, 2048, 1000, 64), (1000, 1024, 2500, 128), (40, 4096, 64, 32), (480, 512, 6144, 64), (270, 256, 6000, 32)])
def test_follows_the_definition(ops, rows, k, ffn, group, x_type, x_group):
    x, xs, w = inputs(ops, rows, k, ffn, group, x_type, x_group, rows + k)
    check(ops.w4_gated(x, w, x_scale=xs, out_dtype=F32), x, xs, w, "silu")
    y = ops.w4_gated(x, w, x_scale=xs, activation="gelu")
    assert y.dtype == (BF16 if x_type in TOP else x_type)
    check(y, x, xs, w, "gelu")


@pytest.mark.parametrize("x_type,x_group", [(BF16, 0), (F16, 0), (E4M3, 0), (I8, 0), (E4M3, 256), (I8, 128)])
@pytest.mark.parametrize("rows,k,ffn,group", [
    (3, 4096, 200, 32), (40, 4096, 200, 128), (2, 1536, 2600, 64), (30, 1536, 2600, 128), (2, 1536, 6144, 128), (70, 2048, 3000, 32),
    (130, 2048, 1000, 64), (300, 1536, 1500, 128), (500, 1536, 6144, 64), (1000, 4096, 1300, 128)])
def test_sums_are_exact_where_they_can_be(ops, rows, k, ffn, group, x_type, x_group):
    """Long sums without a rounding, over every dealing out of K and every width of a tile: what is left is the activation's error."""
    x, xs, codes, scales = exact_gated_case(rows, k, ffn, group, x_type, x_group, rows + k, "cuda")
    w = ops.Int4Weight(codes, scales)
    ref, _ = decode_ref.gated(x, xs, codes, scales, activation="silu")
    out = ops.w4_gated(x, w, x_scale=xs, out_dtype=F32)
    assert ((out.double() - ref).abs() <= exact_gated_limit(ref)).all() and w.status() == 0


@pytest.mark.parametrize("x_type", [BF16, F16, E4M3, I8])
@pytest.mark.parametrize("rows,k,ffn,group", [(1, 32, 1, 32), (5, 64, 7, 64), (70, 96, 128, 32), (130, 160, 20, 32), (2, 1376, 500, 32), (35, 192, 64, 64)])
def test_odd_sizes(ops, rows, k, ffn, group, x_type):
    """k that ends inside a block, fewer outputs than a tile, one row to just above a tile's tokens."""
    x, xs, w = inputs(ops, rows, k, ffn, group, x_type, 0, rows)
    check(ops.w4_gated(x, w, x_scale=xs, out_dtype=F32), x, xs, w, "silu")


@pytest.mark.parametrize("x_type", [BF16, F16, E4M3, I8])
@pytest.mark.parametrize("rows", [2, 40, 200])
def test_every_code_and_every_place(ops, rows, x_type):
    """One x at a time: the outputs are single weights, n - 8 times its scale (gate) and a constant (up)."""
    k, ffn, group = 256, 192, 64
    codes = torch.empty(2 * ffn, k // 2, dtype=torch.uint8)
    n = (torch.arange(ffn)[:, None] * 7 + torch.arange(k) * 3 + torch.arange(k) // 16) % 16
    codes[:ffn] = (n[:, 0::2] | n[:, 1::2] << 4).to(torch.uint8)
    codes[ffn:] = 0x99  # 1
    w = ops.Int4Weight(codes.cuda(), torch.full((2 * ffn, k // group), 0.25, dtype=F16, device="cuda"))
    x = torch.zeros(rows, k, device="cuda")
    at = (torch.arange(rows, device="cuda") * 53) % k
    x[torch.arange(rows, device="cuda"), at] = 8.0
    xs = torch.ones(rows, 1, device="cuda") if x_type in TOP else None
    out = ops.w4_gated(x.to(x_type), w, x_scale=xs, out_dtype=F32)
    g = (n.cuda().double() - 8).t()[at] * 2.0
    ref = g * torch.sigmoid(g) * 2.0
    assert ((out.double() - ref).abs() <= 2.0 ** -19 * ref.abs()).all()


def test_extreme_codes_and_scales(ops):
    """The largest sums that int8 codes can have, gates far out on both sides, scales of 0 and the smallest ones."""
    k, ffn = 2048, 128
    codes = torch.zeros(2 * ffn, k // 2, dtype=torch.uint8, device="cuda")  # all -8
    codes[1::2] = 0xff  # all 7
    scales = torch.full((2 * ffn, k // 128), 2.0 ** -10, dtype=F16, device="cuda")
    scales[2:4], scales[4:6] = 0.0, 2.0 ** -24
    w = ops.Int4Weight(codes, scales)
    for sign in (1, -1):
        for x_type in (I8, E4M3, F16):
            x = torch.full((40, k), 127 * sign if x_type == I8 else 448.0 * sign, device="cuda").to(x_type)
            xs = torch.full((40, 1), 0.25, device="cuda") if x_type in TOP else None
            out = ops.w4_gated(x, w, x_scale=xs, out_dtype=F32)
            check(out, x, xs, w, "silu")
            assert (out[:, 2:4] == 0).all()


@pytest.mark.parametrize("rows,k", [(2, 64), (200, 64), (3, 1024), (40, 1024), (600, 256)])
def test_gates_far_below_zero(ops, rows, k):
    """g and u are exact (one x, codes -8 and 1), exp is good to 2^-21, the sum, the reciprocal and the products to some steps: 2^-20 in
    all; gelu's z is off by six roundings, 6 * 2^-24 |z| < 2^-21 |z|; a reciprocal below the normal numbers, 2^-126, may count as 0."""
    ffn = 128
    codes = torch.zeros(2 * ffn, k // 2, dtype=torch.uint8, device="cuda")
    codes[ffn:] = 0x99
    scales = torch.ones(2 * ffn, k // 32, dtype=F16, device="cuda")
    x = torch.zeros(rows, k, dtype=BF16, device="cuda")
    x[torch.arange(rows, device="cuda"), (torch.arange(rows, device="cuda") * 37) % k] = 1.0
    for activation, ends in (("silu", (10.0, 104.0)), ("gelu", (3.0, 14.0))):
        scales[:ffn] = torch.linspace(*ends, ffn, device="cuda")[:, None].div(8).to(F16)
        w = ops.Int4Weight(codes, scales)
        out = ops.w4_gated(x, w, activation=activation, out_dtype=F32)
        g = scales[:ffn, 0].double() * -8
        z = g if activation == "silu" else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
        ref = g / (1 + torch.exp(-z))
        relative = 2.0 ** -20 + (0 if activation == "silu" else 2.0 ** -21 * z.abs())
        assert ((out.double() - ref).abs() <= relative * ref.abs() + 2.0 ** -126 * g.abs()).all()
        assert (out[:, z > -86] < 0).all()


def test_rows_that_are_not_finite_stay_by_themselves(ops):
    x, _, w = inputs(ops, 40, 512, 200, 128, BF16, 0, 3)
    want = ops.w4_gated(x, w)
    x[7, 100], x[20, 3] = math.nan, math.inf
    got = ops.w4_gated(x, w)
    keep = [i for i in range(40) if i not in (7, 20)]
    assert torch.isnan(got[7]).all() and torch.equal(got[keep], want[keep])
    x, xs, w = inputs(ops, 40, 512, 200, 128, E4M3, 128, 3)
    want = ops.w4_gated(x, w, x_scale=xs)
    xs[7] = math.nan
    got = ops.w4_gated(x, w, x_scale=xs)
    assert torch.isnan(got[7]).all() and torch.equal(got[keep + [20]], want[keep + [20]])


@pytest.mark.parametrize("rows", [1, 20, 100, 400])
def test_rows_of_any_stride_and_place(ops, rows):
    x, _, w = inputs(ops, rows, 256, 136, 64, BF16, 0, rows)
    want = ops.w4_gated(x, w)
    for off, width in ((0, 264), (1, 257), (3, 300), (8, 272)):
        room = torch.full((rows, width), math.nan, dtype=BF16, device="cuda")
        view = room[:, off:off + 256] if off + 256 <= width else None
        if view is None:
            continue
        view.copy_(x)
        place = torch.full((rows + 1, 140), 7.0, dtype=BF16, device="cuda")
        got = ops.w4_gated(view, w, out=place[:rows, 3:139])
        assert torch.equal(got, want) and (place[rows] == 7).all() and (place[:, :3] == 7).all() and (place[:, 139:] == 7).all()


def test_a_row_does_not_depend_on_the_others(ops):
    """Tiles of other widths add up in the same order where K is dealt out the same way: rows of one batch, wherever they stand."""
    x, _, w = inputs(ops, 300, 1024, 256, 128, F16, 0, 5)
    a = ops.w4_gated(x, w)
    order = torch.randperm(300, device="cuda")
    assert torch.equal(ops.w4_gated(x[order].contiguous(), w), a[order])
    assert torch.equal(ops.w4_gated(x, w), a)


def test_graph_streams_and_exchanged_tensors(ops):
    x, xs, w = inputs(ops, 9, 512, 384, 128, E4M3, 0, 6)
    out = ops.w4_gated(x, w, x_scale=xs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.w4_gated(x, w, x_scale=xs)
    y, ys, _ = inputs(ops, 9, 512, 384, 128, E4M3, 0, 7)
    x.copy_(y)
    xs.copy_(ys)
    graph.replay()
    assert torch.equal(held, ops.w4_gated(y, w, x_scale=ys)) and not torch.equal(held, out)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (a, b):
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(20):
        with torch.cuda.stream(a if i % 2 else b):
            got.append(ops.w4_gated(y, w, x_scale=ys))
    torch.cuda.synchronize()
    assert all(torch.equal(g, held) for g in got)
    w.codes = w.codes.flip(0).contiguous()
    check(ops.w4_gated(y, w, x_scale=ys), y, ys, w, "silu")


def test_refusals(ops):
    x, xs, w = inputs(ops, 4, 256, 64, 64, I8, 0, 8)
    h = torch.zeros(4, 256, dtype=BF16, device="cuda")
    odd = ops.Int4Weight(w.codes[:127].contiguous(), w.scales[:127].contiguous())
    assert ops.w4_gated(h[:0], w).shape == (0, 64)
    for bad in (lambda: ops.w4_gated(x, w), lambda: ops.w4_gated(h, w, x_scale=xs), lambda: ops.w4_gated(h.float(), w),
                lambda: ops.w4_gated(h[:, :128], w), lambda: ops.w4_gated(h.cpu(), w), lambda: ops.w4_gated(h, odd),
                lambda: ops.w4_gated(h, w, activation="relu"), lambda: ops.w4_gated(h, w, out_dtype=I8),
                lambda: ops.w4_gated(h, w, out=torch.zeros(4, 63, device="cuda")), lambda: ops.w4_gated(h.t(), w),
                lambda: ops.w4_gated(x, w, x_scale=xs.expand(4, 4).contiguous()),
                lambda: ops.w4_gated(h, w, out=torch.zeros(1, 64, device="cuda").expand(4, 64))):
        with pytest.raises(ValueError):
            bad()


def test_an_output_over_x_is_refused(ops):
    from gemma4_omni_b200._lib import ListenerLibError
    x, _, w = inputs(ops, 9, 256, 128, 64, BF16, 0, 9)
    want = ops.w4_gated(x, w)
    room = torch.zeros(9, 512, dtype=BF16, device="cuda")
    room[:, :256] = x
    for bad in (room[:, :128], room[:, 200:328], room.view(-1)[:9 * 128].view(9, 128), room.view(F32)[:, 64:192]):
        with pytest.raises(ListenerLibError):
            ops.w4_gated(room[:, :256], w, out=bad)
    assert torch.equal(room[:, :256], x)
    assert torch.equal(ops.w4_gated(room[:, :256], w, out=room[:, 256:384]), want)
