"""The entries between a block's products and at its end refuse bad arguments before they touch a GPU."""
from __future__ import annotations

import decimal
import math

import pytest

P = 1 << 20  # a 16-byte aligned address that no call reads


@pytest.fixture(scope="module")
def lib(pkg):
    from gemma4_omni_b200 import _lib, build
    build.build_library()
    return _lib.load()


@pytest.mark.parametrize("name,good,changes", [
    ("lb_op_head_norm_rotary",
     [P, 512, 64, 8, P, 128, 64, 2, 1, 1, 64, P, 0, P, 64, 0, P, P, 0, 1, 1e-6, P, 512, 64, P, 128, 64, None],
     [(0, None), (3, 0), (4, None), (7, -1), (8, 2), (9, 0), (10, 0), (10, 63), (10, 1026), (11, None), (13, None), (14, 66), (14, 31),
      (18, 2), (20, -1.0), (20, math.nan), (21, None), (24, None)]),
    ("lb_op_w4_gated", [P, 256, 1, None, 0, 4, P, P, 64, 100, 256, 0, P, 100, 1, None, None],
     [(0, None), (0, P + 2), (1, 255), (1, 257), (2, 0), (2, 4), (3, P), (4, 128), (5, 0), (6, None), (6, P + 8), (7, None), (8, 16), (8, 256),
      (9, 0), (10, 0), (10, 100), (11, 2), (11, -1), (12, None), (13, 99), (14, 2), (14, 4)]),
    ("lb_op_sample", [P, 100, 1, 2, 100, P, 0, None, 1.0, None, 0, None, 1.0, None, 0.0, P, None, None],
     [(0, None), (1, 99), (2, 2), (2, 7), (3, 0), (4, 0), (5, None), (8, -1.0), (8, math.nan), (8, math.inf), (12, -0.5), (12, math.nan),
      (14, -0.1), (14, 1.5), (14, math.nan), (15, None)]),
])
def test_refusals(lib, name, good, changes):
    for at, value in changes:
        args = list(good)
        args[at] = value
        assert getattr(lib, name)(*args) == -1, (at, value)


Q, K, Y, Z = (i * (P << 8) for i in range(1, 5))  # addresses apart


@pytest.mark.parametrize("name,good,changes", [
    ("lb_op_head_norm_rotary",
     [Q, 640, 64, 8, Q + 1024, 640, 64, 2, 1, 4, 64, P, 0, P, 64, 0, P, P, 0, 1, 1e-6, Y, 512, 64, Z, 128, 64, None],
     # an output over an input in part, over the other one's, over the other output
     [{21: Q + 128}, {21: Q, 22: 512}, {21: Q - 2}, {24: Q}, {24: Q + 1024 + 640 * 2 * 3 + 126}, {21: Q + 1024}, {24: Y + 3 * 1024 + 1022},
      {24: Y, 25: 512}, {21: Q, 22: 640, 24: Q + 1022}, {2: 0, 21: Q, 22: 640, 23: 0, 24: Q, 26: 0}]),
    ("lb_op_w4_gated", [Q, 256, 1, None, 0, 4, P, P, 64, 100, 256, 0, Y, 100, 1, None, None],
     [{12: Q}, {12: Q + 2046}, {12: Q - 799}, {13: 256, 12: Q + 512 - 2}, {13: 256, 12: Q + 256}, {14: 0, 12: Q - 1599}, {5: 1, 12: Q + 511}]),
])
def test_refusals_of_outputs_that_share_memory(lib, name, good, changes):
    for change in changes:
        args = list(good)
        for at, value in change.items():
            args[at] = value
        assert getattr(lib, name)(*args) == -1, change


@pytest.mark.parametrize("name,good,changes", [
    ("lb_op_head_norm_rotary",
     [Q, 512, 64, 8, K, 128, 64, 2, 1, 1, 64, P, 0, P, 64, 0, P, P, 0, 1, 1e-6, Y, 512, 64, Z, 128, 64, None],
     [(0, None), (3, 0), (4, None), (7, -1), (8, 2), (9, 0), (10, 0), (10, 63), (10, 1026), (11, None), (13, None), (14, 66), (14, 31),
      (18, 2), (20, -1.0), (20, math.nan), (21, None), (24, None)]),
    ("lb_op_w4_gated", [Q, 256, 1, None, 0, 4, P, P, 64, 100, 256, 0, Y, 100, 1, None, None],
     [(0, None), (0, Q + 2), (1, 255), (1, 257), (2, 0), (2, 4), (3, P), (4, 128), (5, 0), (6, None), (6, P + 8), (7, None), (8, 16), (8, 256),
      (9, 0), (10, 0), (10, 100), (11, 2), (11, -1), (12, None), (13, 99), (14, 2), (14, 4)]),
])
def test_refusals_of_calls_that_share_no_memory(lib, name, good, changes):
    for at, value in changes:
        args = list(good)
        args[at] = value
        assert getattr(lib, name)(*args) == -1, (at, value)


def test_capacity(lib):
    assert lib.lb_op_sample(P, 300000, 1, 2, 262145, P, 0, None, 1.0, None, 0, None, 1.0, None, 0.0, P, None, None) == -4


def test_turns_are_the_frequencies(pkg):
    """base ** (-2 i / dim) radians as 64-bit fractions of a turn, to 2^-52 of a radian as doubles have them."""
    from gemma4_omni_b200 import decode_ops as ops
    for dim, base in ((64, 10000.0), (256, 1000000.0), (2, 10.0)):
        turns = ops._turns(dim, base)
        assert len(turns) == dim // 2
        for i, t in enumerate(turns):
            assert abs(t / 2.0 ** 64 * 2 * math.pi - base ** (-2.0 * i / dim)) <= 2.0 ** -51


def test_turns_of_large_frequencies(pkg):
    """What is left of the whole turns of any double, over whole numbers (pi by Gauss's formula to 450 digits)."""
    from fractions import Fraction
    from gemma4_omni_b200 import decode_ops as ops
    one = 10 ** 460

    def arctan(n):
        return sum((-1) ** k * (one // n ** (2 * k + 1) // (2 * k + 1)) for k in range(400))

    two_pi = Fraction(2 * (48 * arctan(18) + 32 * arctan(57) - 20 * arctan(239)), one)
    assert abs(float(two_pi) - 2 * math.pi) < 1e-15

    def want(radians):
        v = round(radians * 2 ** 64 / two_pi) % 2 ** 64
        return v - 2 ** 64 if v >= 2 ** 63 else v

    for f in (0.0, 5e-324, 1e-10, 1.0, -1.0, 3.0, 1e15, 1e33, -1e40, 1e80, 2.0 ** 1000, 1.7976931348623157e308, -1.7976931348623157e308):
        assert ops._fraction(decimal.Decimal(f)) == want(Fraction(f)), f
    # a base below 1 has frequencies above it: 1, base ** -1/2
    for base in (0.25, 1e-30, 1e-300):
        root = Fraction(math.isqrt(int(10 ** 800 / Fraction(base))), 10 ** 400)
        assert ops._turns(4, base) == (want(Fraction(1)), want(root))


@pytest.mark.parametrize("k,group", [(1536, 128), (4096, 32)])
def test_exact_gated_case_shows_small_faults(k, group):
    """What the case of exact sums is for: weights rounded to bf16, one column left out, or the scales of two groups or rows exchanged
    leave its bound at most outputs that they touch."""
    import torch
    from helpers import exact_gated_case, exact_gated_limit
    from oracle import decode_ref
    x, _, codes, scales = exact_gated_case(8, k, 64, group, torch.bfloat16, 0, k, "cpu")
    weight = (torch.stack([codes & 15, codes >> 4], 2).view(128, k).double() - 8) * scales.double().repeat_interleave(group, 1)

    def gated(w, x=x.double()):
        g, u = (x @ w.t()).chunk(2, 1)
        return g * torch.sigmoid(g) * u

    ref, _ = decode_ref.gated(x, None, codes, scales, activation="silu")
    assert ((gated(weight) - ref).abs() <= exact_gated_limit(ref) / 2 ** 20).all()
    sums = x.double() @ weight.t()
    assert torch.equal(sums, sums.float().double()) and torch.equal((x.float() @ weight.t().float()).double(), sums)
    short = x.double().clone()
    short[:, k // 2 + 1] = 0
    turned = scales.roll(1, 1).double().repeat_interleave(group, 1)
    rows = scales.roll(1, 0).double().repeat_interleave(group, 1)
    for wrong in (gated(weight.bfloat16().double()), gated(weight, short), gated(weight / scales.double().repeat_interleave(group, 1) * turned),
                  gated(weight / scales.double().repeat_interleave(group, 1) * rows)):
        assert ((wrong - ref).abs() > exact_gated_limit(ref)).double().mean() > 0.9


def test_wrappers_have_no_cpu_path(pkg):
    import torch
    from gemma4_omni_b200 import decode_ops as ops
    with pytest.raises(ValueError):
        ops.Rotary.create(64, device="cpu")
    with pytest.raises(ValueError):
        ops.sample_tokens(torch.zeros(2, 64), torch.zeros(2))
