"""One text-decoder block over the paged 8-bit cache: the consumer of the tower's soft tokens.

``DecoderBlock.step`` runs, for the new tokens of a planned step (``PageDirectory.plan``),

    norm -> q, k, v -> rotary -> cache append -> attention -> output -> norm -> gated feed-forward

with the operators of ``decode_ops``: the norms add the residual and leave 8-bit
codes, the products read those codes against 4-bit weights, keys and values
go to the cache as int8 with a scale per page and head.  With ``DecoderConfig.fused`` the rotation (with norms of queries
and keys for each head, where ``qk_norm`` asks for them) and the gate run in the operators too (``head_norm_rotary``,
``w4_gated``: rounded once), otherwise in plain torch.  ``DecoderHead`` turns the last hidden rows into tokens.  They are a block
and a head as a decoder has them, not a model: weights are given by the caller (``synthetic`` makes seeded ones).
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
    activation: str = "silu"  # or "gelu" (tanh)
    fused: bool = False       # rotation and gate in the operators
    qk_norm: bool = False     # norms of queries and keys for each head (fused)

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
    down [hidden, ffn] as ``Int4Weight``; norm1, norm2 f32 [hidden]; with qk_norm also q_norm, k_norm f32 [head_dim]."""

    def __init__(self, cfg: DecoderConfig, weights: dict):
        self.cfg = cfg
        shapes = {"qkv": (cfg.qkv, cfg.hidden), "out": (cfg.hidden, cfg.heads * cfg.head_dim),
                  "gate_up": (2 * cfg.ffn, cfg.hidden), "down": (cfg.hidden, cfg.ffn)}
        for name, shape in shapes.items():
            w = weights[name]
            if (w.out_features, w.k) != shape:
                raise ValueError(f"{name} must be {shape}")
        if cfg.activation not in ops.ACTIVATIONS:
            raise ValueError(f"activation must be one of {tuple(ops.ACTIVATIONS)}")
        if cfg.qk_norm and not cfg.fused:
            raise ValueError("qk_norm comes with fused")
        for name in ("q_norm", "k_norm") if cfg.qk_norm else ():
            if weights[name].shape != (cfg.head_dim,):
                raise ValueError(f"{name} must be [{cfg.head_dim}]")
        self.w = weights
        self.rotary = ops.Rotary.create(cfg.head_dim, base=cfg.rope_base, device=weights["qkv"].device) if cfg.fused else None

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
        for name in ("q_norm", "k_norm") if cfg.qk_norm else ():
            w[name] = 1.0 + 0.1 * torch.randn(cfg.head_dim, generator=g, device=device)
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
        if c.fused:
            q_norm, k_norm = (self.w["q_norm"], self.w["k_norm"]) if c.qk_norm else (None, None)
            q, k = ops.head_norm_rotary(q, k, at, self.rotary, q_weight=q_norm, k_weight=k_norm, eps=c.rms_eps, norm=c.qk_norm)
        else:
            q, k = rotary(q, at, c.rope_base), rotary(k, at, c.rope_base)
        cache.append(k, v, plan.slots[:t])
        y = ops.kv8_attention(q, cache, plan.row_tables, plan.kv_len, plan.cu_tokens, max_new=max_new,
                              window=c.window, softcap=c.softcap)
        y = ops.w4_matvec(y.view(t, c.heads * c.head_dim), self.w["out"])
        x, xs, h = ops.rms_norm8(y, self.w["norm2"], residual=hidden, eps=c.rms_eps)
        if c.fused:
            y = ops.w4_gated(x, self.w["gate_up"], x_scale=xs, activation=c.activation)
        else:
            gate, up = ops.w4_matvec(x, self.w["gate_up"], x_scale=xs).split(c.ffn, 1)
            y = (torch.nn.functional.silu(gate) if c.activation == "silu" else torch.nn.functional.gelu(gate, approximate="tanh")) * up
        return h + ops.w4_matvec(y, self.w["down"])


class DecoderHead:
    """The end of a decoder: norm, the vocabulary's product, and the draw of a token for each row.  The normed rows are e4m3 with a
    scale a row (``rms_norm8``), as before a block's products: logits of 16-bit rows are the caller's own ``w4_matvec``.
    ``norm`` f32 [hidden], ``vocab`` [vocab, hidden] as ``Int4Weight``."""

    def __init__(self, norm: torch.Tensor, vocab: ops.Int4Weight, *, rms_eps: float = 1e-6):
        if norm.shape != (vocab.k,):
            raise ValueError(f"norm must be [{vocab.k}]")
        self.norm, self.vocab, self.rms_eps = norm, vocab, rms_eps

    @classmethod
    def synthetic(cls, hidden: int, vocab: int, seed: int, device: torch.device | str = "cuda") -> "DecoderHead":
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        w = torch.randn(vocab, hidden, generator=g, device=device) * (2.0 * hidden ** -0.5)
        return cls(1.0 + 0.1 * torch.randn(hidden, generator=g, device=device), ops.Int4Weight.quantize(w))

    def logits(self, hidden: torch.Tensor) -> torch.Tensor:
        """hidden bf16 [rows, hidden] -> float32 [rows, vocab]."""
        x, xs, _ = ops.rms_norm8(hidden, self.norm, eps=self.rms_eps)
        return ops.w4_matvec(x, self.vocab, x_scale=xs, out_dtype=torch.float32)

    def sample(self, hidden: torch.Tensor, uniform: torch.Tensor, **settings):
        """The rows' next tokens, with the given random numbers; ``settings`` and the result as ``sample_tokens`` has them."""
        return ops.sample_tokens(self.logits(hidden), uniform, **settings)
