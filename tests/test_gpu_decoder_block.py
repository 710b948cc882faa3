"""A decoder block through the operators: against the same block in 64 bits from what its weights and
cache stand for, one tick at a time against all at once, and the example that feeds it from the tower."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

from oracle import decode_ref

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def block(pkg):
    from gemma4_omni_b200.decoder_block import DecoderBlock, DecoderConfig
    return DecoderBlock.synthetic(DecoderConfig(hidden=512, heads=8, kv_heads=2, head_dim=64, ffn=1024, softcap=30.0), seed=1)


def directory():
    from gemma4_omni_b200.decode_ops import PageDirectory
    return PageDirectory.create(sessions=4, max_pages=8, pages=32, page_tokens=16)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def run(block, chunks):
    """chunks: for each step, the [tokens, hidden] of every session; the outputs by session."""
    pages = directory()
    cache = block.new_cache(pages.pages, pages.page_tokens)
    outs = [[] for _ in chunks[0]]
    for step in chunks:
        new = [len(c) for c in step]
        plan = pages.plan(ints(list(range(len(step)))), ints(new), max_tokens=sum(new))
        y = block.step(torch.cat(step), plan, cache, max_new=max(new))
        pages.commit(plan)
        for o, part in zip(outs, y.split(new)):
            o.append(part)
    assert cache.status() == 0 and plan.status() == 0
    return [torch.cat(o) for o in outs], pages, cache, plan


def reference(block, x, session, pages, cache):
    """The block on one session's tokens in 64 bits; keys and values are what the cache stands for."""
    c, w = block.cfg, {k: v.dequantize().double() if hasattr(v, "dequantize") else v.double() for k, v in block.w.items()}
    x = x.double()
    n = x.shape[0]
    q = (decode_ref.rms_norm(x, None, w["norm1"], eps=c.rms_eps)[1] @ w["qkv"].t())[:, : c.heads * c.head_dim]
    half = c.head_dim // 2
    a = torch.arange(n, device="cuda").double()[:, None, None] * c.rope_base ** (-torch.arange(half, device="cuda").double() / half)
    q1, q2 = q.view(n, c.heads, c.head_dim).split(half, -1)
    q = torch.cat([q1 * a.cos() - q2 * a.sin(), q2 * a.cos() + q1 * a.sin()], -1)
    y, _, _, _ = decode_ref.attention(q, cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale, pages.tables[session:session + 1],
                                      ints([n]), ints([0, n]), scale=c.head_dim ** -0.5, window=c.window, softcap=c.softcap)
    h = x + y.reshape(n, -1) @ w["out"].t()
    gate, up = (decode_ref.rms_norm(h, None, w["norm2"], eps=c.rms_eps)[1] @ w["gate_up"].t()).split(c.ffn, 1)
    return h + (gate * torch.sigmoid(gate) * up) @ w["down"].t()


def test_block_follows_its_definition(block):
    """Two e4m3 activations (2^-4 each, in the mean a third of it) and bf16 stores: 5 % of the output's norm."""
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    xs = [torch.randn(n, 512, generator=g, device="cuda").to(torch.bfloat16) for n in (37, 1, 64)]
    outs, pages, cache, _ = run(block, [xs])
    for s, (x, y) in enumerate(zip(xs, outs)):
        ref = reference(block, x, s, pages, cache)
        assert (y.double() - ref).norm() <= 0.05 * ref.norm()


def test_ticks_one_by_one_agree_with_a_whole_chunk(block):
    """The keys and values of a page are rounded once more where its scale grows (half a step of 1 / 127 of its
    largest value at most), and 8-bit activations fall on one of two neighbours: 5 % of the output's norm."""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    xs = [torch.randn(40, 512, generator=g, device="cuda").to(torch.bfloat16) for _ in range(3)]
    whole, _, _, _ = run(block, [xs])
    ticks, pages, _, plan = run(block, [[x[2 * t:2 * t + 2] for x in xs] for t in range(20)])
    assert pages.lengths.tolist() == [40, 40, 40, 0] and plan.kv_len.tolist() == [40, 40, 40]
    for a, b in zip(whole, ticks):
        assert (a.double() - b.double()).norm() <= 0.05 * a.double().norm()


def test_sessions_do_not_see_one_another(block):
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    a, b, c = (torch.randn(20, 512, generator=g, device="cuda").to(torch.bfloat16) for _ in range(3))
    one, _, _, _ = run(block, [[a, b]])
    two, _, _, _ = run(block, [[a, c]])
    assert torch.equal(one[0], two[0]) and not torch.equal(one[1], two[1])


def test_example_runs():
    spec = importlib.util.spec_from_file_location("answer_step", ROOT / "examples" / "answer_step.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    result = module.main(ticks=12)
    assert result["status"] == {"tower": 0, "cache": 0, "pages": 0, "plan": 0}
    assert result["lengths"][:4] == [24, 0, 24, 0]
    assert result["out"].shape[0] == 4 and torch.isfinite(result["out"].float()).all()


def test_a_block_of_other_shapes_is_refused(block):
    from gemma4_omni_b200.decoder_block import DecoderBlock, DecoderConfig
    with pytest.raises(ValueError):
        DecoderBlock(DecoderConfig(hidden=512, heads=8, kv_heads=2, head_dim=64, ffn=512), block.w)
