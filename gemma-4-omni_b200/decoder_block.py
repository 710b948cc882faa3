"""One text-decoder block over the paged 8-bit cache: the consumer of the tower's soft tokens.

``DecoderBlock.step`` runs, for the new tokens of a planned step (``PageDirectory.plan``),

    norm -> q, k, v -> rotary -> cache append -> attention -> output -> norm -> gated feed-forward

with the operators of ``decode_ops``: the norms add the residual and leave 8-bit
codes, the products read those codes against 4-bit weights, keys and values
go to the cache as int8 with a scale per page and head.  Rotary embedding and the
gate are plain torch.  It is a block as a decoder has it, not a model: weights are given by the caller
(``DecoderBlock.synthetic`` makes seeded ones).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import decode_ops as ops


@dataclass(frozen=True)
class DecoderConfig:
    hidden: int = 1536
    heads: int = 8
    kv_heads: int = 1
    head_dim: int = 256
    ffn: int = 6144
    window: int = 0
    softcap: float = 0.0
    rope_base: float = 10_000.0
    rms_eps: float = 1e-6
    group: int = 128

    @property
    def qkv(self) -> int:
        return (self.heads + 2 * self.kv_heads) * self.head_dim


def rotary(x: torch.Tensor, positions: torch.Tensor, base: float) -> torch.Tensor:
    """Rotates [tokens, heads, dim] by its positions (halves paired), in 32 bits."""
    half = x.shape[-1] // 2
    inv = base ** (-torch.arange(half, device=x.device, dtype=torch.float32) / half)
    a = positions.float()[:, None, None] * inv
    x1, x2 = x.float().split(half, -1)
    return torch.cat([x1 * a.cos() - x2 * a.sin(), x2 * a.cos() + x1 * a.sin()], -1).to(x.dtype)


class DecoderBlock:
    """``weights``: qkv [qkv, hidden], out [hidden, heads * head_dim], gate_up [2 * ffn, hidden],
    down [hidden, ffn] as ``Int4Weight``; norm1, norm2 f32 [hidden]."""

    def __init__(self, cfg: DecoderConfig, weights: dict):
        self.cfg = cfg
        shapes = {"qkv": (cfg.qkv, cfg.hidden), "out": (cfg.hidden, cfg.heads * cfg.head_dim),
                  "gate_up": (2 * cfg.ffn, cfg.hidden), "down": (cfg.hidden, cfg.ffn)}
        for name, shape in shapes.items():
            w = weights[name]
            if (w.out_features, w.k) != shape:
                raise ValueError(f"{name} must be {shape}")
        self.w = weights

    @classmethod
    def synthetic(cls, cfg: DecoderConfig, seed: int, device: torch.device | str = "cuda") -> "DecoderBlock":
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def matrix(out: int, k: int) -> ops.Int4Weight:
            return ops.Int4Weight.quantize(torch.randn(out, k, generator=g, device=device) * k ** -0.5, group=cfg.group)

        w = {"qkv": matrix(cfg.qkv, cfg.hidden), "out": matrix(cfg.hidden, cfg.heads * cfg.head_dim),
             "gate_up": matrix(2 * cfg.ffn, cfg.hidden), "down": matrix(cfg.hidden, cfg.ffn)}
        for name in ("norm1", "norm2"):
            w[name] = 1.0 + 0.1 * torch.randn(cfg.hidden, generator=g, device=device)
        return cls(cfg, w)

    def new_cache(self, pages: int, page_tokens: int, device: torch.device | str = "cuda") -> ops.Kv8Cache:
        return ops.Kv8Cache.create(pages=pages, kv_heads=self.cfg.kv_heads, page_tokens=page_tokens, dim=self.cfg.head_dim,
                                   device=device)

    def step(self, hidden: torch.Tensor, plan: ops.PagePlan, cache: ops.Kv8Cache, *, max_new: int) -> torch.Tensor:
        """hidden bf16 [tokens, hidden] of the plan's tokens, in order -> the block's output, bf16."""
        c = self.cfg
        t = hidden.shape[0]
        x, xs, _ = ops.rms_norm8(hidden, self.w["norm1"], eps=c.rms_eps)
        q, k, v = ops.w4_matvec(x, self.w["qkv"], x_scale=xs).view(t, c.heads + 2 * c.kv_heads, c.head_dim).split(
            (c.heads, c.kv_heads, c.kv_heads), 1)
        at = plan.positions[:t]
        cache.append(rotary(k, at, c.rope_base), v, plan.slots[:t])
        y = ops.kv8_attention(rotary(q, at, c.rope_base), cache, plan.row_tables, plan.kv_len, plan.cu_tokens, max_new=max_new,
                              window=c.window, softcap=c.softcap)
        y = ops.w4_matvec(y.view(t, c.heads * c.head_dim), self.w["out"])
        x, xs, h = ops.rms_norm8(y, self.w["norm2"], residual=hidden, eps=c.rms_eps)
        gate, up = ops.w4_matvec(x, self.w["gate_up"], x_scale=xs).split(c.ffn, 1)
        return h + ops.w4_matvec(torch.nn.functional.silu(gate) * up, self.w["down"])
