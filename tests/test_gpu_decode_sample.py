"""Sampling against the rule over Python numbers.  Tokens are whole numbers and have to be equal: masses of the kernel
and of the rule differ by a unit of 2^-45 at most where a rounding of exp falls the other way, so a row of 10^5
tokens whose random number lies within 10^5 * 2^-45 of a border is one in a million.  Log probabilities are off by their
rounding, 2^-24 relative, and by the masses' units."""
from __future__ import annotations

import math
import random

import pytest
import torch

from oracle import decode_ref

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops(pkg):
    from gemma4_omni_b200 import decode_ops
    return decode_ops


def logits_of(rows, vocab, dtype, seed, spread=2.5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, device="cuda") * spread
    x[:, :: max(1, vocab // 7)] += 6.0
    u = torch.rand(rows, generator=g, device="cuda")
    return x.to(dtype), u


def check(ops, x, u, **settings):
    tokens, logprobs = ops.sample_tokens(x, u, return_logprobs=True, **settings)
    assert tokens.dtype == torch.int64 and logprobs.dtype == torch.float32
    for r in range(x.shape[0]):
        own = {k: (float(v[r]) if k != "top_k" else int(v[r])) if isinstance(v, torch.Tensor) else
               (v if k == "top_k" else float(torch.tensor(v, dtype=F32))) for k, v in settings.items()}
        own.setdefault("temperature", 1.0)
        token, logprob = decode_ref.sample(x[r], float(u[r]), **own)
        assert int(tokens[r]) == token, (r, own)
        if logprob == -math.inf:
            assert float(logprobs[r]) == logprob
        else:
            assert abs(float(logprobs[r]) - logprob) <= 2.0 ** -23 * abs(logprob) + 1e-9
    return tokens


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=50, top_p=0.95), dict(top_k=1), dict(top_k=700),
            dict(top_p=0.9), dict(top_p=0.999, temperature=1.5), dict(min_p=0.05), dict(top_k=2000, top_p=0.97, min_p=0.001),
            dict(top_p=0.0), dict(temperature=40.0, top_p=0.5), dict(temperature=40.0, top_k=3000), dict(temperature=1e-6),
            dict(temperature=1e-3, top_k=5, top_p=0.5, min_p=1.0)]


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("rows,vocab,dtype", [(3, 1, F32), (4, 7, BF16), (3, 512, F16), (3, 513, BF16), (3, 2049, F32), (2, 16384, BF16),
                                              (2, 16387, F16), (2, 32003, F16), (2, 65537, F32), (2, 131072, BF16), (1, 262144, F32)])
def test_follows_the_rule(ops, rows, vocab, dtype, settings):
    x, u = logits_of(rows, vocab, dtype, vocab + len(settings))
    check(ops, x, u, **settings)


@pytest.mark.parametrize("vocab", [300, 5000, 40000, 131072])
@pytest.mark.parametrize("values", [1, 2, 5, 300])
def test_equal_logits_are_cut_by_index(ops, vocab, values):
    """Few values, each many times: cuts fall between tokens of one value."""
    g = torch.Generator(device="cuda")
    g.manual_seed(values)
    x = torch.randint(0, values, (2, vocab), generator=g, device="cuda").float() * 0.25 - 3.0
    u = torch.tensor([0.999, 0.31], device="cuda")
    for settings in (dict(top_k=vocab // 3), dict(top_p=0.4), dict(top_k=vocab // 2, top_p=0.7), dict(top_k=vocab - 1), dict(top_k=3, top_p=0.5),
                     dict(min_p=0.9), dict()):
        check(ops, x, u, **settings)


def test_one_part_in_many_values(ops):
    """So many different values so near one another that a bin is divided more than once."""
    n = 100000
    x = (1.0 + torch.arange(n, device="cuda").float() * 2.0 ** -23)[torch.randperm(n, device="cuda")].view(1, n)
    x = torch.cat([x, x * 2.0 ** -126, -x])  # also tiny values, and falling bit patterns
    u = torch.tensor([0.2, 0.77, 0.5], device="cuda")
    for settings in (dict(top_k=33333), dict(top_p=0.3), dict(top_k=70000, top_p=0.77), dict(temperature=100.0, top_p=0.123)):
        check(ops, x, u, **settings)


def test_masked_rows_and_infinities(ops):
    x, u = logits_of(8, 40000, F32, 3)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, :39999] = -math.inf
    x[3, 100:] = math.nan
    x[4, 5], x[4, 39000], x[4, 7] = math.inf, math.inf, math.nan
    x[5] = torch.finfo(F32).min
    x[6, 1:] = -math.inf
    x[7] = x[7].abs() * 0.0  # zeros of both signs are equal
    x[7, ::2] = -0.0
    for settings in (dict(), dict(top_k=1000), dict(top_p=0.6), dict(top_k=50, top_p=0.9, min_p=0.1), dict(temperature=0.0)):
        tokens = check(ops, x, u, **settings)
        assert tokens[:3].tolist() == [-1, -1, 39999] and int(tokens[4]) in (5, 39000)
    small = torch.tensor([[-math.inf, 1.0, math.nan, 1.0], [-math.inf] * 4], device="cuda")
    for settings in (dict(), dict(top_k=1), dict(top_p=0.1), dict(top_k=3)):
        check(ops, small, torch.tensor([0.9, 0.9], device="cuda"), **settings)


@pytest.mark.parametrize("vocab", [300, 5000, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_the_lowest_numbers(ops, vocab, dtype):
    """Rows that a mask filled with the type's lowest number, beside -inf and NaN, which have no mass at any temperature."""
    lowest = torch.finfo(dtype).min
    near = torch.tensor([lowest], dtype=dtype, device="cuda")
    ups = [near]
    for _ in range(5):
        ups.append(torch.nextafter(ups[-1], torch.zeros_like(near)))
    x = torch.full((6, vocab), -math.inf, dtype=dtype, device="cuda")
    x[0, ::3] = lowest
    x[1], x[1, 1::2] = lowest, math.nan
    x[2, vocab - 2] = lowest
    x[3, 5::7], x[3, 6::7] = lowest, ups[1]
    for i, v in enumerate(ups):
        x[4, i::11] = v
    x[5], x[5, 7] = lowest, ups[1]
    u = torch.tensor([0.999, 0.5, 0.9, 0.3, 0.999999, 0.7], device="cuda")
    for settings in (dict(), dict(top_k=100), dict(top_p=0.6), dict(top_k=vocab - 10, top_p=0.9, min_p=0.1), dict(min_p=0.5),
                     dict(temperature=0.0), dict(temperature=1e-6), dict(temperature=1e30), dict(temperature=1e30, top_p=0.5),
                     dict(temperature=1e30, top_k=vocab // 2, top_p=0.999999)):
        tokens = check(ops, x, u, **settings)
        assert int(tokens[2]) == vocab - 2


@pytest.mark.parametrize("vocab", [400, 2000, 32003, 70001])
@pytest.mark.parametrize("dtype,mask", [(F32, torch.finfo(F32).min), (F32, torch.finfo(BF16).min), (F32, -1e38), (F32, -1e37), (BF16, torch.finfo(BF16).min),
                                        (BF16, -2e37), (F16, torch.finfo(F16).min)])
def test_top_k_among_masked_tokens(ops, vocab, dtype, mask):
    """Fewer tokens than top_k asks for, the rest of a mask's large finite value or -inf: cuts fall among tokens without a mass, whose
    distance to the maximum, in bins, is a number or not."""
    g = torch.Generator(device="cuda")
    g.manual_seed(vocab)
    rows = [(60, 10), (60, 200), (vocab - 5, 5), (vocab // 2, vocab // 3), (1, vocab - 1)]
    x = torch.full((len(rows), vocab), -math.inf, dtype=dtype, device="cuda")
    for row, (live, masked) in zip(x, rows):
        order = torch.randperm(vocab, generator=g, device="cuda")
        row[order[:live]] = (torch.randn(live, generator=g, device="cuda") * 2.5).to(dtype)
        row[order[live:live + masked]] = mask
    u = torch.tensor([0.9999, 0.5, 0.3, 0.99, 0.7], device="cuda")
    k = torch.tensor([live + (masked + 1) // 2 for live, masked in rows], dtype=torch.int32, device="cuda")
    for temperature in (0.8, 1.0, 1.3, 10.0):
        check(ops, x, u, temperature=temperature, top_k=k)
        check(ops, x, u, temperature=temperature, top_k=k, top_p=0.95, min_p=0.01)
    check(ops, x, u, top_p=0.9999)
    check(ops, x, u, top_k=64, top_p=1.0 - 2.0 ** -24)


def vectorised(x, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The rule over many rows at once, on the GPU: (tokens, log probabilities)."""
    x, order = torch.sort(x.float(), dim=1, descending=True, stable=True)
    t32 = [float(torch.tensor(v, dtype=F32)) for v in (temperature, top_p, min_p)]
    mass = torch.round(torch.exp((x.double() - x[:, :1].double()) / t32[0]) * 2.0 ** 45).to(torch.int64)
    if top_k:
        mass[:, top_k:] = 0
    upto = mass.cumsum(1)
    if t32[1] < 1.0:
        mass[upto - mass >= torch.ceil(t32[1] * upto[:, -1:].double()).to(torch.int64).clamp(min=1)] = 0
    mass[mass < math.ceil(t32[2] * 2.0 ** 45)] = 0
    mass = torch.zeros_like(mass).scatter_(1, order, mass)
    upto = mass.cumsum(1)
    total = upto[:, -1:]
    target = torch.minimum(torch.floor(u.double()[:, None] * total.double()).to(torch.int64), total - 1)
    token = torch.searchsorted(upto, target, right=True)
    return token[:, 0], torch.log(mass.gather(1, token).double() / total.double())[:, 0]


@pytest.mark.parametrize("settings", [dict(top_p=0.999, temperature=1.5), dict(top_p=0.9), dict(top_p=0.5, temperature=2.0),
                                      dict(top_p=0.7, temperature=0.6), dict(top_k=3000), dict(top_k=20000, top_p=0.9),
                                      dict(top_k=600, top_p=0.99, min_p=0.01), dict(min_p=0.001, temperature=3.0)])
@pytest.mark.parametrize("vocab,dtype", [(262144, F32), (131072, F32), (131072, BF16), (20001, F32)])
def test_cuts_in_every_place(ops, vocab, dtype, settings):
    """Cuts deep in a row's bulk, 48 rows each: a token that one pass sees in another bin than the next pass moves a
    cut by some ranks, which is 10^-6 of a total, so the totals are held to 10^-7 (the log's rounding and some)."""
    x, u = logits_of(48, vocab, dtype, vocab)
    tokens, logprobs = ops.sample_tokens(x, u, return_logprobs=True, **settings)
    want, log = vectorised(x, u, **settings)
    assert torch.equal(tokens, want)
    assert ((logprobs.double() - log).abs() <= 2.0 ** -24 * log.abs() + 1e-9).all()


def test_settings_by_row_and_64_bit_numbers(ops):
    rng = random.Random(4)
    x, _ = logits_of(40, 20000, BF16, 8)
    u = torch.tensor([rng.random() for _ in range(38)] + [0.0, 1.0 - 2.0 ** -53], dtype=torch.float64, device="cuda")

    def column(values, dtype):
        return torch.tensor([rng.choice(values) for _ in range(40)], dtype=dtype, device="cuda")

    check(ops, x, u, temperature=column([0.0, 0.5, 1.0, 2.0], F32), top_k=column([0, 1, 40, 600, 30000], torch.int32),
          top_p=column([0.0, 0.3, 0.95, 1.0, 2.0], F32), min_p=column([0.0, 0.01, 0.5, 1.0], F32))
    # out of range: as the nearer one that is in it
    odd = ops.sample_tokens(x, u, temperature=torch.full((40,), -1.0, device="cuda"))
    assert torch.equal(odd, ops.sample_tokens(x, u, temperature=0.0))
    odd = ops.sample_tokens(x, u, top_k=torch.full((40,), -5, dtype=torch.int32, device="cuda"),
                            top_p=torch.full((40,), math.nan, device="cuda"), min_p=torch.full((40,), math.nan, device="cuda"))
    assert torch.equal(odd, ops.sample_tokens(x, u))
    assert torch.equal(ops.sample_tokens(x, u, min_p=torch.full((40,), 7.0, device="cuda")), ops.sample_tokens(x, u, min_p=1.0))
    for wild, tame in ((-1.0, 0.0), (math.nan, 0.0), (5.0, 1.0 - 2.0 ** -53)):
        a, b = (torch.full((40,), v, dtype=torch.float64, device="cuda") for v in (wild, tame))
        assert torch.equal(ops.sample_tokens(x, a), ops.sample_tokens(x, b))


def test_strides_alignment_and_many_rows(ops):
    """Rows apart by any number of elements, from any address; more rows than run at once."""
    room = torch.zeros(300, 2100, dtype=BF16, device="cuda")
    x, u = logits_of(300, 2053, BF16, 9)
    for off in (0, 1, 3, 7):
        view = room[:, off:off + 2053]
        view.copy_(x)
        got = check(ops, view, u, top_k=100, top_p=0.9) if off == 3 else ops.sample_tokens(view, u, top_k=100, top_p=0.9)
        assert torch.equal(got, ops.sample_tokens(x, u, top_k=100, top_p=0.9))
    x, u = logits_of(600, 50001, F16, 10)
    tokens = ops.sample_tokens(x, u, top_p=0.8)
    some = [0, 1, 299, 598, 599]
    assert tokens[some].tolist() == [decode_ref.sample(x[r], float(u[r]), temperature=1.0, top_p=float(torch.tensor(0.8)))[0] for r in some]
    assert torch.equal(tokens, ops.sample_tokens(x, u, top_p=0.8))


def test_frequencies_of_draws(ops):
    """Even steps of u give each token its probability to within one step a border."""
    p = torch.tensor([0.5, 0.25, 0.125, 0.0625, 0.0625], device="cuda")
    n = 4096
    x = p.log().expand(n, 5)
    u = (torch.arange(n, device="cuda").double() + 0.5) / n
    tokens = ops.sample_tokens(x.contiguous(), u)
    count = torch.bincount(tokens, minlength=5)
    assert (count - p * n).abs().max() <= 1 and (tokens.diff() >= 0).all()


def test_graph_and_streams(ops):
    x, u = logits_of(5, 131072, BF16, 11)
    graph = torch.cuda.CUDAGraph()
    ops.sample_tokens(x, u, top_p=0.9)
    with torch.cuda.graph(graph):
        out = ops.sample_tokens(x, u, top_p=0.9)
    for seed in (12, 13):
        y, v = logits_of(5, 131072, BF16, seed)
        x.copy_(y)
        u.copy_(v)
        graph.replay()
        assert torch.equal(out, ops.sample_tokens(y, v, top_p=0.9))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    want = ops.sample_tokens(x, u, top_k=900)
    for s in (a, b):
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(10):
        with torch.cuda.stream(a if i % 2 else b):
            got.append(ops.sample_tokens(x, u, top_k=900))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_refusals(ops):
    x, u = logits_of(4, 100, F32, 1)
    assert ops.sample_tokens(x[:0], u[:0]).shape == (0,)
    ones = torch.ones(4, device="cuda")
    for bad in (lambda: ops.sample_tokens(x.double(), u), lambda: ops.sample_tokens(x[0], u), lambda: ops.sample_tokens(x, u[:3]),
                lambda: ops.sample_tokens(x, u.half()), lambda: ops.sample_tokens(x, u.cpu()), lambda: ops.sample_tokens(x.cpu(), u.cpu()),
                lambda: ops.sample_tokens(x.t(), u), lambda: ops.sample_tokens(x[:1].expand(4, 100), u),
                lambda: ops.sample_tokens(x, u, temperature=-0.1), lambda: ops.sample_tokens(x, u, temperature=math.nan),
                lambda: ops.sample_tokens(x, u, temperature=math.inf), lambda: ops.sample_tokens(x, u, top_k=-1),
                lambda: ops.sample_tokens(x, u, top_p=-0.5), lambda: ops.sample_tokens(x, u, min_p=1.5),
                lambda: ops.sample_tokens(x, u, temperature=ones.double()), lambda: ops.sample_tokens(x, u, top_k=ones),
                lambda: ops.sample_tokens(x, u, top_p=ones[:2]),
                lambda: ops.sample_tokens(torch.zeros(1, 262145, device="cuda"), u[:1])):
        with pytest.raises(ValueError):
            bad()
