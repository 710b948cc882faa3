"""Text-decoder operators: paged 8-bit K/V cache, its attention, 8-bit norm, 4-bit matvec.

The audio tower ends at two soft tokens per session and tick.  Their consumer, the
text decoder, keeps a private and growing K/V cache per session (reference:
native/gemma4_listener/gemma4_listener_cache.cu:34-42, duplex_kernel/kv_cache.py:40-80).
Here the caches of all sessions share one pool of pages:

- ``PageDirectory``: which pages a session has.  ``plan`` maps a step's new tokens
  to pages and cache slots on the GPU, ``commit`` installs the plan, ``release``
  gives a session's pages back.  Like the packer, a plan changes nothing
  until it is committed, and the k-th page needed is the k-th lowest free page.
- ``Kv8Cache``: int8 keys and values with one scale per page and kv head;
  ``append`` writes the planned tokens, ``kv8_attention`` reads them.
- ``rms_norm8``: residual addition + RMS norm with an 8-bit output and scales.
- ``Int4Weight`` / ``w4_matvec``: products with 4-bit weights and group scales.
- ``Rotary`` / ``head_norm_rotary``: norms of queries and keys for each head, with the position rotation.
- ``w4_gated``: both projections of a gated feed-forward block, the activation and the product.
- ``sample_tokens``: the next tokens from logits and given random numbers.

Every call is enqueued on torch's current stream of the tensors' device and can be
captured into a CUDA graph; none synchronises except the ``status`` reads.
There is no CPU path.
"""
from __future__ import annotations

import decimal
import functools
import math
from dataclasses import dataclass

import torch

from . import _lib

DTYPE_CODES = {torch.float32: _lib.LB_F32, torch.bfloat16: _lib.LB_BF16, torch.int8: _lib.LB_I8,
               torch.float16: _lib.LB_F16, torch.float8_e4m3fn: _lib.LB_E4M3}
FLOAT_INPUTS = (torch.float32, torch.bfloat16, torch.float16)
HEAD_DIMS = (64, 128, 256)
PAGE_TOKENS_MAX = 256
MAX_PLAN_ROWS = 8192
MAX_SESSIONS = 262144
MAX_PLAN_TOKENS = 1 << 26
INT32_MAX = (1 << 31) - 1
MAX_HEAD_DIM = 1024
MAX_VOCAB = 262144


def _call(device: torch.device, name: str, *args) -> None:
    """Runs one C entry on the current stream of ``device`` (appended to the arguments)."""
    fn = getattr(_lib.load(), name)
    # the raw handle of torch.cuda.current_stream(device), without an object around it
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    else:
        rc = fn(*args, stream)
    if rc != _lib.LB_OK:
        _lib.check(name, rc)


def _need(t: torch.Tensor, name: str, dtype, shape: tuple, device: torch.device) -> None:
    """Refuses what is not a contiguous tensor of this type and shape on this device."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on {device}")


def _row_step(t: torch.Tensor) -> int:
    """Elements between the rows of a 2-D tensor (of a single row: its width, whatever stride it has); 0 where
    a row's elements are not neighbours or rows overlap."""
    rows, cols = t.shape
    if cols > 1 and rows and t.stride(1) != 1:
        return 0
    step = t.stride(0) if rows > 1 else cols
    return step if step >= cols else 0


def _spread(t: torch.Tensor) -> bool:
    """Whether the values of a 3-D tensor lie apart: heads within tokens, or tokens within heads."""
    (n, heads, dim), (a, b, _) = t.shape, t.stride()
    a, b = a if n > 1 else heads * dim * max(b, 1), b if heads > 1 else dim
    return (b >= dim and a >= (heads - 1) * b + dim) or (n > 1 and a >= dim and b >= (n - 1) * a + dim)


def _exchangeable(name: str, dtype: torch.dtype, shape, align: int = 1) -> property:
    """An attribute that holds a tensor.  It may be exchanged for another one of the same type, ``shape(owner)``
    and device, whose address the next call takes; anything else is refused when it is set."""
    slot = "_t_" + name

    def get(self) -> torch.Tensor:
        return getattr(self, slot)

    def put(self, t: torch.Tensor) -> None:
        _need(t, name, dtype, shape(self), self.device)
        if t.data_ptr() % align:
            raise ValueError(f"{name} must be {align}-byte aligned")
        setattr(self, slot, t)

    return property(get, put)


def _cuda(device: torch.device, what: str) -> torch.device:
    if device.type != "cuda":
        raise ValueError(f"{what} runs on a CUDA device (no CPU fallback)")
    return device  # of a tensor: it has an index


@dataclass
class PagePlan:
    """One step's pages: what ``Kv8Cache.append`` and ``kv8_attention`` read."""
    sessions: torch.Tensor    # int32 [n], the plan's own copy
    row_tables: torch.Tensor  # int32 [n, max_pages], -1 past a row's last page
    kv_len: torch.Tensor      # int32 [n], tokens of the session after the step
    cu_tokens: torch.Tensor   # int32 [n + 1]
    slots: torch.Tensor       # int64 [max_tokens], -1 past the last token
    positions: torch.Tensor   # int32 [max_tokens]
    token_rows: torch.Tensor  # int32 [max_tokens]
    status_word: torch.Tensor  # int32 [1]

    def status(self) -> int:
        """LB_DEV_* bits of a refused plan or of a commit that came too late, 0 of a good one (synchronises)."""
        return int(self.status_word.item())


class PageDirectory:
    """The pages of every session: ``tables`` int32 [sessions, max_pages], ``lengths``
    int32 [sessions], ``used`` int32 words with one bit per page."""

    tables = _exchangeable("tables", torch.int32, lambda d: (d.sessions, d.max_pages))
    lengths = _exchangeable("lengths", torch.int32, lambda d: (d.sessions,))
    used = _exchangeable("used", torch.int32, lambda d: (-(-d.pages // 32),))

    def __init__(self, tables: torch.Tensor, lengths: torch.Tensor, used: torch.Tensor, *, pages: int,
                 page_tokens: int):
        self.device = _cuda(tables.device, "PageDirectory")
        if tables.dim() != 2 or not 0 < tables.shape[0] <= MAX_SESSIONS or tables.shape[1] < 1:
            raise ValueError(f"tables must be [sessions, max_pages] with at most {MAX_SESSIONS} sessions")
        if page_tokens % 16 or not 16 <= page_tokens <= PAGE_TOKENS_MAX:
            raise ValueError(f"page_tokens must be a multiple of 16, at most {PAGE_TOKENS_MAX}")
        if pages < 1:
            raise ValueError("pages must be positive")
        self.sessions, self.max_pages = (int(v) for v in tables.shape)
        if self.max_pages * page_tokens >= 2 ** 31:
            raise ValueError("a session holds fewer than 2^31 tokens")
        self.pages, self.page_tokens = int(pages), int(page_tokens)
        self.tables, self.lengths, self.used = tables, lengths, used
        self._released = torch.zeros(1, dtype=torch.int32, device=self.device)

    @classmethod
    def create(cls, *, sessions: int, max_pages: int, pages: int, page_tokens: int,
               device: torch.device | str = "cuda") -> "PageDirectory":
        """An empty directory: every page is free."""
        return cls(torch.full((sessions, max_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(sessions, dtype=torch.int32, device=device),
                   torch.zeros(-(-pages // 32), dtype=torch.int32, device=device), pages=pages,
                   page_tokens=page_tokens)

    def plan(self, sessions: torch.Tensor, new_tokens: torch.Tensor, *, max_tokens: int) -> PagePlan:
        """Plans a step that adds ``new_tokens[i]`` tokens to ``sessions[i]`` (distinct).

        ``max_tokens``: the rows of the step's token tensors; the plan is refused if
        the counts sum to more.  The directory is not changed."""
        n, dev = sessions.numel(), self.device
        if not 0 < n <= MAX_PLAN_ROWS:
            raise ValueError(f"a plan has between 1 and {MAX_PLAN_ROWS} rows")
        if not 0 < max_tokens <= MAX_PLAN_TOKENS:
            raise ValueError(f"max_tokens must be between 1 and {MAX_PLAN_TOKENS}")
        _need(sessions, "sessions", torch.int32, (n,), dev)
        _need(new_tokens, "new_tokens", torch.int32, (n,), dev)
        # one allocation: the 64-bit slots, then the 32-bit arrays
        mp = self.max_pages
        words = 2 * max_tokens, n * mp, max_tokens, max_tokens, n, n + 1, n, 1
        buf = self._t_lengths.new_empty(sum(words))
        slots, tables, positions, rows, kv_len, cu, planned, status = buf.split(words)
        p_slots = buf.data_ptr()
        p_tables = p_slots + 8 * max_tokens
        p_pos = p_tables + 4 * n * mp
        p_rows = p_pos + 4 * max_tokens
        p_len = p_rows + 4 * max_tokens
        p_cu = p_len + 4 * n
        p_planned = p_cu + 4 * n + 4
        _call(dev, "lb_plan_step", n, sessions.data_ptr(), new_tokens.data_ptr(), self.sessions, mp, self.pages,
              self.page_tokens, self._t_tables.data_ptr(), self._t_lengths.data_ptr(), self._t_used.data_ptr(), max_tokens,
              p_tables, p_len, p_cu, p_slots, p_pos, p_rows, p_planned, p_planned + 4 * n)
        return PagePlan(planned, tables.view(n, mp), kv_len, cu, slots.view(torch.int64), positions, rows, status)

    def commit(self, plan: PagePlan) -> None:
        """Installs a plan.  One that was refused, or that no longer fits the directory (another plan
        was committed or a session released since), changes nothing; the latter gets
        LB_DEV_STALE_COMMIT in its ``status``."""
        n = plan.sessions.numel()
        for name, shape in (("sessions", (n,)), ("row_tables", (n, self.max_pages)), ("kv_len", (n,)), ("cu_tokens", (n + 1,)),
                            ("status_word", (1,))):
            _need(getattr(plan, name), name, torch.int32, shape, self.device)
        _call(self.device, "lb_commit_step", n, plan.sessions.data_ptr(), self.sessions, self.max_pages, self.pages,
              self.page_tokens, plan.row_tables.data_ptr(), plan.kv_len.data_ptr(), plan.cu_tokens.data_ptr(),
              plan.status_word.data_ptr(), self._t_tables.data_ptr(), self._t_lengths.data_ptr(), self._t_used.data_ptr())

    def release(self, sessions: torch.Tensor) -> None:
        """Gives the pages of these distinct sessions back."""
        n = sessions.numel()
        _need(sessions, "sessions", torch.int32, (n,), self.device)
        if n:
            _call(self.device, "lb_release_pages", n, sessions.data_ptr(), self.sessions, self.max_pages, self.pages,
                  self.page_tokens, self._t_tables.data_ptr(), self._t_lengths.data_ptr(), self._t_used.data_ptr(),
                  self._released.data_ptr())

    def status(self) -> int:
        """LB_DEV_* bits of the releases so far (synchronises)."""
        return int(self._released.item())


class Kv8Cache:
    """Keys and values as int8 codes [pages, kv_heads, page_tokens, dim] with one f32
    scale per page and head [pages, kv_heads]: value = code * scale."""

    k_codes = _exchangeable("k_codes", torch.int8, lambda c: (c.pages, c.kv_heads, c.page_tokens, c.dim), 16)
    v_codes = _exchangeable("v_codes", torch.int8, lambda c: (c.pages, c.kv_heads, c.page_tokens, c.dim), 16)
    k_scale = _exchangeable("k_scale", torch.float32, lambda c: (c.pages, c.kv_heads))
    v_scale = _exchangeable("v_scale", torch.float32, lambda c: (c.pages, c.kv_heads))
    status_word = _exchangeable("status_word", torch.int32, lambda c: (1,))

    def __init__(self, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        self.device = _cuda(k_codes.device, "Kv8Cache")
        if k_codes.dim() != 4 or 0 in k_codes.shape:
            raise ValueError("codes must be [pages, kv_heads, page_tokens, dim]")
        self.pages, self.kv_heads, self.page_tokens, self.dim = (int(v) for v in k_codes.shape)
        if self.page_tokens % 16 or self.page_tokens > PAGE_TOKENS_MAX:
            raise ValueError(f"page_tokens must be a multiple of 16, at most {PAGE_TOKENS_MAX}")
        if self.dim not in HEAD_DIMS:
            raise ValueError(f"dim must be one of {HEAD_DIMS}")
        self.k_codes, self.v_codes, self.k_scale, self.v_scale = k_codes, v_codes, k_scale, v_scale
        self.status_word = torch.zeros(1, dtype=torch.int32, device=self.device)

    @classmethod
    def create(cls, *, pages: int, kv_heads: int, page_tokens: int, dim: int,
               device: torch.device | str = "cuda") -> "Kv8Cache":
        shape = (pages, kv_heads, page_tokens, dim)
        return cls(torch.zeros(shape, dtype=torch.int8, device=device), torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.zeros(shape[:2], device=device), torch.zeros(shape[:2], device=device))

    def _pointers(self) -> tuple[int, int, int, int]:
        # (past the properties, which cost as much as the addresses)
        return (self._t_k_codes.data_ptr(), self._t_v_codes.data_ptr(), self._t_k_scale.data_ptr(),
                self._t_v_scale.data_ptr())

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Writes k, v [tokens, kv_heads, dim] to ``slots`` int64 [tokens] (negative: skipped).

        The tokens of one page follow one another in order, as a ``PagePlan`` has
        them, with no skipped one between: those after a gap are not written and set
        LB_DEV_SPLIT_PAGE in ``status``.  A page's scale only grows; the codes it held are rounded to the new scale."""
        n = slots.numel()
        if k.dtype not in FLOAT_INPUTS or v.dtype != k.dtype:
            raise ValueError("k and v must both be float32, bfloat16 or float16")
        for name, t in (("k", k), ("v", v)):
            if t.shape != (n, self.kv_heads, self.dim) or t.device != self.device or t.stride(2) != 1:
                raise ValueError(f"{name} must be [{n}, {self.kv_heads}, {self.dim}] on {self.device}, its rows contiguous")
        _need(slots, "slots", torch.int64, (n,), self.device)
        if n == 0:
            return
        kc, vc, ks, vs = self._pointers()
        _call(self.device, "lb_op_kv8_append", k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
              v.stride(1), DTYPE_CODES[k.dtype], n, self.kv_heads, self.dim, slots.data_ptr(), kc, vc, ks, vs,
              self.pages, self.page_tokens, self._t_status_word.data_ptr())

    def status(self) -> int:
        """LB_DEV_* bits seen by appends and attention so far (synchronises)."""
        return int(self.status_word.item())


@functools.lru_cache(maxsize=None)
def _workspace(dim: int, heads: int, kv_heads: int, max_new: int) -> int:
    return _lib.load().lb_kv8_attention_workspace(dim, heads, kv_heads, max_new)


def kv8_attention(q: torch.Tensor, cache: Kv8Cache, row_tables: torch.Tensor, kv_len: torch.Tensor,
                  cu_tokens: torch.Tensor, *, max_new: int, scale: float | None = None, window: int = 0,
                  softcap: float = 0.0, out: torch.Tensor | None = None, return_lse: bool = False):
    """Causal attention of a step's tokens over the cache (which already holds them).

    q [tokens, heads, dim] bfloat16 / float16; row r has the tokens
    [cu_tokens[r], cu_tokens[r+1]), the last of its kv_len[r].  ``max_new``: the most
    tokens of a row (a hint for the work's split, never for what is computed).
    ``scale`` defaults to dim ** -0.5; ``window`` > 0 keeps the last ``window`` keys;
    ``softcap`` > 0 squashes scores with softcap * tanh(score / softcap).  A token that sees no key gets
    zeros.  Returns out [tokens, heads, dim], or (out, lse f32 [tokens, heads])."""
    dev = cache.device
    if q.dim() != 3 or q.shape[2] != cache.dim or q.device != dev or (q.numel() and q.stride(2) != 1):
        raise ValueError(f"q must be [tokens, heads, {cache.dim}] on {dev}, its rows contiguous")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("q must be bfloat16 or float16")
    t, heads, dim = q.shape
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError("heads must be a positive multiple of the cache's kv_heads")
    if row_tables.dim() != 2 or row_tables.shape[0] < 1:
        raise ValueError("row_tables must be [rows, max_pages]")
    n, max_pages = row_tables.shape
    _need(row_tables, "row_tables", torch.int32, (n, max_pages), dev)
    _need(kv_len, "kv_len", torch.int32, (n,), dev)
    _need(cu_tokens, "cu_tokens", torch.int32, (n + 1,), dev)
    if window < 0 or not 0.0 <= softcap < float("inf") or max_new < 1:
        raise ValueError("window and softcap must not be negative, softcap finite, max_new positive")
    if out is None:
        out = q.new_empty(q.shape)
    else:
        _need(out, "out", q.dtype, (t, heads, dim), dev)
    lse = cache._t_k_scale.new_empty((t, heads)) if return_lse else None
    if t:
        kc, vc, ks, vs = cache._pointers()
        space = cache._t_k_codes.new_empty(_workspace(dim, heads, cache.kv_heads, min(max_new, INT32_MAX)))
        _call(dev, "lb_op_kv8_attention", q.data_ptr(), q.stride(0), q.stride(1), DTYPE_CODES[q.dtype], t, n, heads,
              cache.kv_heads, dim, kc, vc, ks, vs, cache.pages, cache.page_tokens, row_tables.data_ptr(), max_pages,
              kv_len.data_ptr(), cu_tokens.data_ptr(), min(max_new, INT32_MAX),
              dim ** -0.5 if scale is None else scale, min(window, INT32_MAX), softcap,
              out.data_ptr(), lse.data_ptr() if return_lse else None, cache._t_status_word.data_ptr(),
              space.data_ptr())
    return (out, lse) if return_lse else out


def rms_norm8(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None, eps: float = 1e-6,
              group: int = 0, dtype: torch.dtype = torch.float8_e4m3fn):
    """(codes [rows, dim] of ``dtype``, scales f32 [rows, dim / group or 1], hidden).

    hidden = x + residual in x's type (x itself without a residual); codes * scales =
    hidden / rms(hidden) * weight.  ``dtype``: float8_e4m3fn or int8; ``group``: columns
    that share a scale, 0 for one scale a row."""
    if x.dim() != 2 or x.dtype not in FLOAT_INPUTS:
        raise ValueError("x must be a float32, bfloat16 or float16 [rows, dim] tensor")
    x_step = _row_step(x)
    if not x_step and x.numel():
        raise ValueError("x's rows must be contiguous and apart")
    dev = _cuda(x.device, "rms_norm8")
    rows, dim = x.shape
    if not 0 < dim <= 16384 or group < 0 or (group and dim % group):
        raise ValueError("dim must be at most 16384 and a multiple of group")
    if dtype not in (torch.float8_e4m3fn, torch.int8):
        raise ValueError("codes are float8_e4m3fn or int8")
    if weight.dtype not in (torch.float32, x.dtype):
        raise ValueError("weight must be float32 or of x's type")
    _need(weight, "weight", weight.dtype, (dim,), dev)
    r_step = 0
    if residual is not None:
        if residual.dtype != x.dtype or residual.shape != x.shape or residual.device != dev:
            raise ValueError("residual must be like x")
        r_step = _row_step(residual)
        if not r_step and rows:
            raise ValueError("residual's rows must be contiguous and apart")
    codes = torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format)
    n_groups = dim // group if group else 1
    scales = (weight.new_empty((rows, n_groups)) if weight.dtype == torch.float32
              else torch.empty((rows, n_groups), dtype=torch.float32, device=dev))
    hidden = x if residual is None else x.new_empty(x.shape)
    if rows:
        _call(dev, "lb_op_rms_norm8", x.data_ptr(), x_step, None if residual is None else residual.data_ptr(),
              r_step, DTYPE_CODES[x.dtype], weight.data_ptr(),
              DTYPE_CODES[weight.dtype], rows, dim, eps, group, DTYPE_CODES[dtype], codes.data_ptr(), scales.data_ptr(),
              None if residual is None else hidden.data_ptr())
    return codes, scales, hidden


class Int4Weight:
    """A [out, k] matrix of 4-bit codes: uint8 [out, k / 2] (low four bits: even k),
    f16 scales [out, k / group]; weight = (code - 8) * scale."""

    codes = _exchangeable("codes", torch.uint8, lambda w: (w.out_features, w.k // 2), 16)
    scales = _exchangeable("scales", torch.float16, lambda w: (w.out_features, w.k // w.group))
    status_word = _exchangeable("status_word", torch.int32, lambda w: (1,))

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        self.device = _cuda(codes.device, "Int4Weight")
        if codes.dim() != 2 or scales.dim() != 2 or 0 in codes.shape or 0 in scales.shape:
            raise ValueError("codes must be [out, k / 2] and scales [out, k / group]")
        self.out_features, self.k = int(codes.shape[0]), 2 * int(codes.shape[1])
        self.group = self.k // int(scales.shape[1])
        if self.group not in (32, 64, 128) or self.group * int(scales.shape[1]) != self.k:
            raise ValueError("groups must have 32, 64 or 128 columns")
        self.codes, self.scales = codes, scales
        self.status_word = torch.zeros(1, dtype=torch.int32, device=self.device)

    def status(self) -> int:
        """LB_DEV_* bits of the gated products so far (synchronises)."""
        return int(self.status_word.item())

    @classmethod
    def quantize(cls, weight: torch.Tensor, group: int = 128) -> "Int4Weight":
        """Rounds a [out, k] matrix to codes -8..7 with scales max |w| / 7 per group."""
        out, k = (int(v) for v in weight.shape)
        if group not in (32, 64, 128) or k % group:
            raise ValueError("groups must have 32, 64 or 128 columns and divide k")
        w = weight.float().view(out, k // group, group)
        scales = (w.abs().amax(2) / 7.0).to(torch.float16)
        s = scales.float()[:, :, None]
        codes = torch.where(s > 0, torch.round(w / s), 0.0).clamp(-8, 7).add(8).to(torch.uint8).view(out, k)
        return cls((codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous(), scales.contiguous())

    def dequantize(self) -> torch.Tensor:
        """The matrix the codes stand for, float32 [out, k]."""
        both = torch.stack([self.codes & 15, self.codes >> 4], 2).view(self.out_features, -1, self.group)
        return ((both.float() - 8.0) * self.scales.float()[:, :, None]).view(self.out_features, self.k)


def _product_input(x: torch.Tensor, weight: Int4Weight, x_scale: torch.Tensor | None) -> tuple[int, int, int]:
    """(rows, columns of a group of x_scale or 0, elements between rows) of a product's x."""
    dev = weight.device
    if x.dim() != 2 or x.shape[1] != weight.k or x.device != dev:
        raise ValueError(f"x must be [rows, {weight.k}] on {dev}")
    rows, group, x_step = int(x.shape[0]), 0, _row_step(x)
    if not x_step and rows:
        raise ValueError("x's rows must be contiguous and apart")
    if x.dtype in (torch.int8, torch.float8_e4m3fn):
        if x_scale is None or x_scale.dim() != 2 or x_scale.shape[1] < 1 or weight.k % x_scale.shape[1]:
            raise ValueError("8-bit x needs x_scale [rows, groups]")
        _need(x_scale, "x_scale", torch.float32, (rows, int(x_scale.shape[1])), dev)
        group = weight.k // int(x_scale.shape[1])
        if group == weight.k:
            group = 0
        elif group % 128:
            raise ValueError("groups of x must have a multiple of 128 columns")
    elif x.dtype not in (torch.bfloat16, torch.float16) or x_scale is not None:
        raise ValueError("x must be bfloat16 or float16 without x_scale, or float8_e4m3fn / int8 with it")
    return rows, group, x_step


def w4_matvec(x: torch.Tensor, weight: Int4Weight, *, x_scale: torch.Tensor | None = None,
              out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [rows, k] times the transposed weight -> [rows, out].

    x is bfloat16 / float16, or float8_e4m3fn / int8 codes with ``x_scale`` f32
    [rows, groups] as ``rms_norm8`` returns them (one group a row, or groups of a
    multiple of 128 columns).  ``out_dtype`` defaults to x's type, bfloat16 for 8-bit x."""
    dev = weight.device
    rows, group, x_step = _product_input(x, weight, x_scale)
    if out is None:
        out_dtype = out_dtype or (x.dtype if x_scale is None else torch.bfloat16)
        if out_dtype not in FLOAT_INPUTS:
            raise ValueError("out_dtype must be float32, bfloat16 or float16")
        out = torch.empty((rows, weight.out_features), dtype=out_dtype, device=dev)
        out_step = weight.out_features
    else:
        if out.dtype not in FLOAT_INPUTS or out.shape != (rows, weight.out_features) or out.device != dev:
            raise ValueError(f"out must be [{rows}, {weight.out_features}] on {dev}")
        out_step = _row_step(out)
        if not out_step and rows:
            raise ValueError("out's rows must be contiguous and apart")
    if rows:
        _call(dev, "lb_op_w4_matvec", x.data_ptr(), x_step, DTYPE_CODES[x.dtype],
              None if x_scale is None else x_scale.data_ptr(), group, rows, weight._t_codes.data_ptr(),
              weight._t_scales.data_ptr(), weight.group, weight.out_features, weight.k, out.data_ptr(), out_step,
              DTYPE_CODES[out.dtype])
    return out


ACTIVATIONS = {"silu": 0, "gelu": 1}


def w4_gated(x: torch.Tensor, weight: Int4Weight, *, x_scale: torch.Tensor | None = None, activation: str = "silu",
             out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """The first half of a gated feed-forward block: act(x gate^T) * (x up^T) -> [rows, ffn], in one kernel.

    ``weight`` [2 * ffn, k] has the gate's rows, then those of up.  x and ``x_scale`` as in ``w4_matvec``, from one row
    to thousands; both products, the activation ("silu", or "gelu" in its tanh form) and the product are in 32
    bits, rounded once.  ``out_dtype`` defaults to x's type, bfloat16 for 8-bit x.  ``out`` shares no memory with x."""
    dev = weight.device
    rows, group, x_step = _product_input(x, weight, x_scale)
    if weight.out_features % 2:
        raise ValueError("weight must have as many rows for the gate as for up")
    ffn = weight.out_features // 2
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}")
    if out is None:
        out_dtype = out_dtype or (x.dtype if x_scale is None else torch.bfloat16)
        if out_dtype not in FLOAT_INPUTS:
            raise ValueError("out_dtype must be float32, bfloat16 or float16")
        out = torch.empty((rows, ffn), dtype=out_dtype, device=dev)
        out_step = ffn
    else:
        if out.dtype not in FLOAT_INPUTS or out.shape != (rows, ffn) or out.device != dev:
            raise ValueError(f"out must be [{rows}, {ffn}] on {dev}")
        out_step = _row_step(out)
        if not out_step and rows:
            raise ValueError("out's rows must be contiguous and apart")
    if rows:
        size = x.element_size()
        if x.data_ptr() % 16 or (rows > 1 and x_step * size % 16):  # rows that TMA cannot address are laid out anew
            x, x_step = x.new_empty(x.shape).copy_(x), weight.k
        _call(dev, "lb_op_w4_gated", x.data_ptr(), x_step, DTYPE_CODES[x.dtype], None if x_scale is None else x_scale.data_ptr(),
              group, rows, weight._t_codes.data_ptr(), weight._t_scales.data_ptr(), weight.group, ffn, weight.k,
              ACTIVATIONS[activation], out.data_ptr(), out_step, DTYPE_CODES[out.dtype], weight._t_status_word.data_ptr())
    return out


_DIGITS = 400  # the 309 before the point of the largest double, 64 bits behind it, and some to spare


@functools.lru_cache(maxsize=1)
def _two_pi() -> decimal.Decimal:
    """2 pi to more than _DIGITS digits, over whole numbers: pi / 4 = 4 arctan(1 / 5) - arctan(1 / 239) (Machin)."""
    one = 10 ** (_DIGITS + 20)

    def arctan(n: int) -> int:
        term = total = one // n
        k = 1
        while term:
            term //= -n * n
            k += 2
            total += term // k
        return total

    with decimal.localcontext() as c:
        c.prec = _DIGITS + 20
        return decimal.Decimal(8 * (4 * arctan(5) - arctan(239))) / one


@functools.lru_cache(maxsize=64)
def _turns(rotary_dim: int, base: float) -> tuple[int, ...]:
    """The frequencies base ** (-2 i / rotary_dim), in turns a position, as signed 64-bit fractions of a turn."""
    with decimal.localcontext() as c:
        c.prec = 50 if base >= 1.0 else _DIGITS  # (digits before the point too)
        return tuple(_fraction(decimal.Decimal(base) ** (decimal.Decimal(-2 * i) / rotary_dim)) for i in range(rotary_dim // 2))


def _fraction(radians: decimal.Decimal) -> int:
    """radians / (2 pi) modulo 1 as a whole number of 2^-64, in the range of int64."""
    with decimal.localcontext() as c:
        c.prec = _DIGITS
        v = int((radians / _two_pi() * 2 ** 64).to_integral_value(decimal.ROUND_HALF_EVEN)) % 2 ** 64
    return v - 2 ** 64 if v >= 2 ** 63 else v


class Rotary:
    """The frequencies of a position rotation of heads of ``dim`` values.

    ``turns`` int64 [rotary_dim / 2]: frequencies in turns a position, as 64-bit fractions, of which no whole turns are left
    over; an angle is good to 2e-9 radians and 2e-19 times the position (2e-7 at 2^40).  ``pairs``: "halves" pairs value i with i + rotary_dim / 2, "neighbours" 2 i with 2 i + 1;
    values from rotary_dim on are not rotated."""

    turns = _exchangeable("turns", torch.int64, lambda r: (r.rotary_dim // 2,), 8)

    def __init__(self, turns: torch.Tensor, dim: int, *, pairs: str = "halves"):
        self.device = _cuda(turns.device, "Rotary")
        if turns.dim() != 1 or turns.shape[0] < 1:
            raise ValueError("turns must be [rotary_dim / 2]")
        self.dim, self.rotary_dim = int(dim), 2 * int(turns.shape[0])
        if self.dim % 2 or not self.rotary_dim <= self.dim <= MAX_HEAD_DIM:
            raise ValueError(f"dim must be even, at most {MAX_HEAD_DIM}, and no less than rotary_dim")
        if pairs not in ("halves", "neighbours"):
            raise ValueError('pairs are "halves" or "neighbours"')
        self.pairs = pairs
        self.turns = turns

    @classmethod
    def create(cls, dim: int, *, rotary_dim: int | None = None, base: float = 10_000.0, pairs: str = "halves",
               device: torch.device | str = "cuda") -> "Rotary":
        """Frequencies base ** (-2 i / rotary_dim) radians a position."""
        rotary_dim = dim if rotary_dim is None else rotary_dim
        if rotary_dim < 2 or rotary_dim % 2 or not 0.0 < base < math.inf:
            raise ValueError("rotary_dim must be even and positive, base positive")
        return cls(torch.tensor(_turns(rotary_dim, float(base)), dtype=torch.int64, device=device), dim, pairs=pairs)

    @classmethod
    def from_frequencies(cls, frequencies, dim: int, *, pairs: str = "halves", device: torch.device | str = "cuda") -> "Rotary":
        """Given frequencies (a sequence of floats or a tensor), in radians a position."""
        values = [float(f) for f in frequencies]
        if not all(math.isfinite(f) for f in values):
            raise ValueError("frequencies must be finite")
        return cls(torch.tensor([_fraction(decimal.Decimal(f)) for f in values], dtype=torch.int64, device=device), dim, pairs=pairs)


def head_norm_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, rotary: Rotary, *,
                     q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                     norm: bool = True, q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """Norms of queries and keys for each head, and their rotation by ``positions``, in one pass: (q, k).

    q [tokens, heads, dim], k [tokens, kv_heads, dim] (or None) of one type, such as views of one product's output; positions
    int32 or int64 [tokens], as a ``PagePlan`` has them.  With ``norm`` each head's values become x / sqrt(mean(x^2) + eps) *
    weight (weights f32 or of q's type, None: 1).  ``q_out`` / ``k_out`` may be q and k themselves, and share
    no memory with an input or one another otherwise (the call is refused)."""
    dev = rotary.device
    if q.dim() != 3 or q.dtype not in FLOAT_INPUTS:
        raise ValueError("q must be a float32, bfloat16 or float16 [tokens, heads, dim] tensor")
    t, heads, dim = q.shape
    if dim != rotary.dim or heads < 1:
        raise ValueError(f"heads have {rotary.dim} values")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64")
    _need(positions, "positions", positions.dtype, (t,), dev)
    if not 0.0 <= eps < math.inf:
        raise ValueError("eps must not be negative")
    q_out, q_args, q_to = _head_side("q", q, q_out, q_weight, dev, norm)
    if k is None:
        if k_out is not None or k_weight is not None:
            raise ValueError("k_out and k_weight come with k")
        kv_heads, k_args, k_to = 0, (None, 0, 0), (None, 0, 0)
    else:
        if k.dim() != 3 or k.dtype != q.dtype or k.shape[0] != t or k.shape[2] != dim:
            raise ValueError("k must be like q but for its number of heads")
        kv_heads = k.shape[1]
        k_out, k_args, k_to = _head_side("k", k, k_out, k_weight, dev, norm)
    weight = q_weight if q_weight is not None else k_weight
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("weights must be of one type")
    if t:
        _call(dev, "lb_op_head_norm_rotary", *q_args, heads, *k_args, kv_heads, DTYPE_CODES[q.dtype],
              t, dim, positions.data_ptr(), positions.dtype == torch.int64, rotary._t_turns.data_ptr(), rotary.rotary_dim,
              rotary.pairs == "neighbours", None if q_weight is None else q_weight.data_ptr(),
              None if k_weight is None else k_weight.data_ptr(), _lib.LB_F32 if weight is None else DTYPE_CODES[weight.dtype], norm, eps,
              *q_to, *k_to)
    return q_out, k_out


def _head_side(name: str, x: torch.Tensor, out: torch.Tensor | None, weight: torch.Tensor | None, dev: torch.device, norm: bool):
    """Checks one of q and k; (its output, address and strides of the input, of the output)."""
    step = x.stride()
    if x.device != dev or (step[2] != 1 and x.numel()):
        raise ValueError(f"{name} must be on {dev}, its rows contiguous")
    if weight is not None:
        if not norm:
            raise ValueError("weights belong to the norm")
        if weight.dtype not in (torch.float32, x.dtype):
            raise ValueError("weights must be float32 or of q's type")
        _need(weight, f"{name}_weight", weight.dtype, (x.shape[2],), dev)
    if out is None:
        out = torch.empty_like(x)  # (of a part of a product's output: contiguous)
        to = out.stride()
    else:
        to = out.stride()
        if out.shape != x.shape or out.dtype != x.dtype or out.device != dev or (out.numel() and (to[2] != 1 or not _spread(out))):
            raise ValueError(f"{name}_out must be like {name}, its rows contiguous and apart")
        if out.data_ptr() == x.data_ptr() and to != step and out.numel():
            raise ValueError(f"{name}_out must have {name}'s strides where it is {name}")
    return out, (x.data_ptr(), step[0], step[1]), (out.data_ptr(), to[0], to[1])


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                  return_logprobs: bool = False):
    """Draws a token a row from ``logits`` [rows, vocab] with the given random numbers ``uniform`` [rows] in [0, 1).

    ``temperature`` (0: the likeliest token), ``top_k`` (0: all), ``top_p`` (1: all) and ``min_p`` (0: all) are numbers, or tensors
    with one for each row (float32; top_k int32).  top_k keeps the first tokens by falling logit (the lower index first),
    top_p of those the first whose probabilities reach top_p, min_p those of at least min_p times the largest
    probability; the token is the first by index at which the sum of what is kept exceeds ``uniform`` times its total.
    Masses are whole numbers of 2^-45 of the largest, so that a result depends on no order of summation.
    Returns int64 [rows] (-1 where a row has nothing to draw: all -inf or NaN), with ``return_logprobs`` also
    float32 [rows], the logarithm of the token's part in what was kept."""
    if logits.dim() != 2 or logits.dtype not in FLOAT_INPUTS:
        raise ValueError("logits must be a float32, bfloat16 or float16 [rows, vocab] tensor")
    dev = _cuda(logits.device, "sample_tokens")
    rows, vocab = logits.shape
    if not 0 < vocab <= MAX_VOCAB:
        raise ValueError(f"a row has between 1 and {MAX_VOCAB} logits")
    step = _row_step(logits)
    if not step and rows:
        raise ValueError("the rows of logits must be contiguous and apart")
    if uniform.dtype not in (torch.float32, torch.float64):
        raise ValueError("uniform must be float32 or float64")
    _need(uniform, "uniform", uniform.dtype, (rows,), dev)
    settings = []
    for name, value, dtype, low, high in (("temperature", temperature, torch.float32, 0.0, 1e30), ("top_k", top_k, torch.int32, 0, math.inf),
                                          ("top_p", top_p, torch.float32, 0.0, math.inf), ("min_p", min_p, torch.float32, 0.0, 1.0)):
        if isinstance(value, torch.Tensor):
            _need(value, name, dtype, (rows,), dev)
            settings += [value.data_ptr(), 0]
        else:
            if not low <= value <= high:
                raise ValueError(f"{name} must be between {low} and {high}")
            settings += [None, min(value, vocab) if dtype == torch.int32 else value]
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)
    logprobs = torch.empty(rows, dtype=torch.float32, device=dev) if return_logprobs else None
    if rows:
        _call(dev, "lb_op_sample", logits.data_ptr(), step, DTYPE_CODES[logits.dtype], rows, vocab, uniform.data_ptr(),
              uniform.dtype == torch.float64, *settings, tokens.data_ptr(), logprobs.data_ptr() if return_logprobs else None)
    return (tokens, logprobs) if return_logprobs else tokens
