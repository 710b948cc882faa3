"""A decoder block that runs all of its step in the operators, and the head that draws tokens from it: against the same block
in 64 bits from what its weights and cache stand for, one tick at a time against all at once, and a captured loop that writes an
answer."""
from __future__ import annotations

import importlib.util
import math
from dataclasses import replace
from pathlib import Path

import pytest
import torch

from oracle import decode_ref

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def parts(pkg):
    from gemma4_omni_b200 import decoder_block
    return decoder_block


def config(parts, **changes):
    return replace(parts.DecoderConfig(hidden=512, heads=8, kv_heads=2, head_dim=64, ffn=1024, softcap=30.0, fused=True), **changes)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def rows(seed, *lengths):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [torch.randn(n, 512, generator=g, device="cuda").to(torch.bfloat16) for n in lengths]


def run(block, chunks):
    """chunks: for each step, the [tokens, hidden] of every session; the outputs by session."""
    from gemma4_omni_b200.decode_ops import PageDirectory
    pages = PageDirectory.create(sessions=4, max_pages=8, pages=32, page_tokens=16)
    cache = block.new_cache(pages.pages, pages.page_tokens)
    outs = [[] for _ in chunks[0]]
    for step in chunks:
        new = [len(c) for c in step]
        plan = pages.plan(ints(list(range(len(step)))), ints(new), max_tokens=sum(new))
        y = block.step(torch.cat(step), plan, cache, max_new=max(new))
        pages.commit(plan)
        for o, part in zip(outs, y.split(new)):
            o.append(part)
    assert cache.status() == 0 and plan.status() == 0 and block.w["gate_up"].status() == 0
    return [torch.cat(o) for o in outs], pages, cache


def reference(block, x, session, pages, cache):
    c, w = block.cfg, {k: v.dequantize().double() if hasattr(v, "dequantize") else v.double() for k, v in block.w.items()}
    x, n = x.double(), x.shape[0]
    q = (decode_ref.rms_norm(x, None, w["norm1"], eps=c.rms_eps)[1] @ w["qkv"].t())[:, : c.heads * c.head_dim]
    freqs = [c.rope_base ** (-2.0 * i / c.head_dim) for i in range(c.head_dim // 2)]
    q = decode_ref.head_norm_rotary(q.view(n, c.heads, c.head_dim), w.get("q_norm"), torch.arange(n, device="cuda"), freqs, rotary=c.head_dim,
                                    pairs="halves", eps=c.rms_eps, norm=c.qk_norm)
    y, _, _, _ = decode_ref.attention(q, cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale, pages.tables[session:session + 1],
                                      ints([n]), ints([0, n]), scale=c.head_dim ** -0.5, window=c.window, softcap=c.softcap)
    h = x + y.reshape(n, -1) @ w["out"].t()
    gate, up = (decode_ref.rms_norm(h, None, w["norm2"], eps=c.rms_eps)[1] @ w["gate_up"].t()).split(c.ffn, 1)
    z = gate if c.activation == "silu" else 2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)
    return h + (gate * torch.sigmoid(z) * up) @ w["down"].t()


@pytest.mark.parametrize("changes", [dict(), dict(qk_norm=True, activation="gelu"), dict(qk_norm=True, window=20, rope_base=1e6)])
def test_block_follows_its_definition(parts, changes):
    """Two e4m3 activations (2^-4 each, in the mean a third of it) and bf16 stores: 5 % of the output's norm."""
    block = parts.DecoderBlock.synthetic(config(parts, **changes), seed=1)
    xs = rows(2, 37, 1, 64)
    outs, pages, cache = run(block, [xs])
    for s, (x, y) in enumerate(zip(xs, outs)):
        ref = reference(block, x, s, pages, cache)
        assert (y.double() - ref).norm() <= 0.05 * ref.norm()


def test_agrees_with_the_block_in_plain_torch(parts):
    """The same weights without the fused parts: q, k and the gate are rounded to bf16 at other places, then meet e4m3 and int8 steps."""
    for activation in ("silu", "gelu"):
        fused = parts.DecoderBlock.synthetic(config(parts, activation=activation), seed=3)
        plain = parts.DecoderBlock(replace(fused.cfg, fused=False), fused.w)
        xs = rows(4, 33, 40)
        a, _, _ = run(fused, [xs])
        b, _, _ = run(plain, [xs])
        for x, y in zip(a, b):
            assert (x.double() - y.double()).norm() <= 0.05 * y.double().norm()


def test_head_norms_weights_count_with_qk_norm_only(parts):
    """A dict of weights that also holds head norms serves a block without them, as it does where rotation and gate are plain torch."""
    normed = parts.DecoderBlock.synthetic(config(parts, qk_norm=True), seed=13)
    cfg = replace(normed.cfg, qk_norm=False)
    xs = rows(14, 20, 3)
    a, _, _ = run(parts.DecoderBlock(cfg, normed.w), [xs])
    b, _, _ = run(parts.DecoderBlock(cfg, {k: v for k, v in normed.w.items() if k not in ("q_norm", "k_norm")}), [xs])
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_ticks_one_by_one_agree_with_a_whole_chunk(parts):
    """As for the block in plain torch: 5 % of the output's norm."""
    block = parts.DecoderBlock.synthetic(config(parts, qk_norm=True), seed=5)
    xs = rows(6, 40, 40, 40)
    whole, _, _ = run(block, [xs])
    ticks, pages, _ = run(block, [[x[2 * t:2 * t + 2] for x in xs] for t in range(20)])
    assert pages.lengths.tolist() == [40, 40, 40, 0]
    for a, b in zip(whole, ticks):
        assert (a.double() - b.double()).norm() <= 0.05 * a.double().norm()


def test_head_draws_by_the_rule_from_its_logits(parts):
    head = parts.DecoderHead.synthetic(512, 5000, seed=7)
    hidden, = rows(8, 9)
    u = torch.rand(9, device="cuda")
    logits = head.logits(hidden)
    y = decode_ref.rms_norm(hidden, None, head.norm, eps=1e-6)[1]
    ref = y @ head.vocab.dequantize().double().t()
    assert (logits.double() - ref).norm() <= 0.05 * ref.norm()  # e4m3 activations
    tokens, logprobs = head.sample(hidden, u, temperature=0.7, top_k=40, top_p=0.9, return_logprobs=True)
    for r in range(9):
        token, logprob = decode_ref.sample(logits[r], float(u[r]), temperature=float(torch.tensor(0.7)), top_k=40, top_p=float(torch.tensor(0.9)))
        assert int(tokens[r]) == token and abs(float(logprobs[r]) - logprob) <= 2.0 ** -23 * abs(logprob) + 1e-9


def test_captured_loop_writes_the_same_answer(parts):
    """Plan, block, head, commit and the next embedding in one graph, replayed: the tokens of the loop that runs call by call."""
    from gemma4_omni_b200.decode_ops import PageDirectory
    block = parts.DecoderBlock.synthetic(config(parts, qk_norm=True), seed=9)
    head = parts.DecoderHead.synthetic(512, 3001, seed=10)
    table = torch.randn(3001, 512, device="cuda").to(torch.bfloat16)
    who, one = ints([2, 0, 3]), ints([1, 1, 1])
    uniform = torch.rand(12, 3, device="cuda")

    def fresh():
        pages = PageDirectory.create(sessions=4, max_pages=4, pages=12, page_tokens=16)
        return pages, block.new_cache(pages.pages, pages.page_tokens), torch.tensor([5, 6, 7], device="cuda"), torch.zeros(3, device="cuda")

    def step(pages, cache, tokens, u):
        plan = pages.plan(who, one, max_tokens=3)
        y = block.step(table[tokens], plan, cache, max_new=1)
        tokens.copy_(head.sample(y, u, temperature=0.9, top_k=200, top_p=0.95))
        pages.commit(plan)

    pages, cache, tokens, u = fresh()
    want = []
    for row in uniform:
        u.copy_(row)
        step(pages, cache, tokens, u)
        want.append(tokens.tolist())
    pages, cache, tokens, u = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(pages, cache, tokens, u)
    got = []
    for row in uniform:
        u.copy_(row)
        graph.replay()
        got.append(tokens.tolist())
    assert got == want and pages.lengths.tolist() == [12, 0, 12, 12] and cache.status() == 0
    assert len({tuple(t) for t in got}) > 3


def test_refusals(parts):
    good = parts.DecoderBlock.synthetic(config(parts, qk_norm=True), seed=11)
    for changes in (dict(activation="relu"), dict(fused=False), dict(head_dim=128, heads=4, kv_heads=1)):
        with pytest.raises(ValueError):
            parts.DecoderBlock(replace(good.cfg, **changes), good.w)
    with pytest.raises(ValueError):
        parts.DecoderHead(torch.ones(100, device="cuda"), good.w["out"])


def test_example_draws_tokens():
    spec = importlib.util.spec_from_file_location("answer_step", ROOT / "examples" / "answer_step.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    # (the tower's split sums are added up in any order, so two runs' soft tokens may differ in their last bits)
    tokens = module.main(ticks=4)["tokens"]
    assert len(tokens) == 2 and all(0 <= t < 1000 for t in tokens)


def test_offsets_beyond_32_bits(pkg):
    """Rows 2^31 elements apart: queries, logits and the gated product's output, beside the same rows close together."""
    from gemma4_omni_b200 import decode_ops as ops
    room = torch.zeros((1 << 31) + (1 << 14), dtype=torch.bfloat16, device="cuda")

    def far(cols):
        return room.as_strided((2, cols), (1 << 31, 1))

    g = torch.Generator(device="cuda")
    g.manual_seed(12)
    near = torch.randn(2, 4096, generator=g, device="cuda").to(torch.bfloat16)
    at, r = torch.tensor([3, 70000], device="cuda"), ops.Rotary.create(128)
    far(1024).copy_(near[:, :1024])
    q = far(1024).unflatten(1, (8, 128))
    want = ops.head_norm_rotary(near[:, :1024].unflatten(1, (8, 128)), None, at, r)[0]
    assert torch.equal(ops.head_norm_rotary(q, None, at, r)[0], want)
    ops.head_norm_rotary(q, None, at, r, q_out=q)
    assert torch.equal(q, want)
    far(4096).copy_(near)
    u = torch.tensor([0.3, 0.8], device="cuda")
    assert torch.equal(ops.sample_tokens(far(4096), u, top_p=0.9), ops.sample_tokens(near, u, top_p=0.9))
    w = ops.Int4Weight.quantize(torch.randn(600, 256, generator=g, device="cuda"))
    x = near[:, :256].contiguous()
    want = ops.w4_gated(x, w)
    ops.w4_gated(x, w, out=far(300))
    assert torch.equal(far(300), want)
    far(256).copy_(x)
    assert torch.equal(ops.w4_gated(far(256), w), want)
