"""The text-decoder operators from their definitions, in 64 bits (torch doubles, any device).

Each function also returns what its callers need to bound a kernel's rounding:
sums of absolute values beside the sums themselves."""
from __future__ import annotations

import math

import torch


def plan(sessions, new, tables, lengths, used, *, page_tokens, max_tokens):
    """The page rule in plain Python over lists: row tables, lengths, tokens' slots / positions / rows, or None if refused."""
    if len(set(sessions)) != len(sessions) or any(s < 0 or s >= len(lengths) for s in sessions):
        return None
    if any(m < 0 for m in new) or sum(new) > max_tokens:
        return None
    width = len(tables[0])
    free = iter([p for p, u in enumerate(used) if not u])
    rows, lens, slots, positions, owner = [], [], [], [], []
    for i, (s, m) in enumerate(zip(sessions, new)):
        held = -(-lengths[s] // page_tokens)
        need = -(-(lengths[s] + m) // page_tokens)
        if need > width:
            return None
        table = list(tables[s][:held])
        for _ in range(need - held):
            page = next(free, None)
            if page is None:
                return None
            table.append(page)
        for t in range(lengths[s], lengths[s] + m):
            slots.append(table[t // page_tokens] * page_tokens + t % page_tokens)
            positions.append(t)
            owner.append(i)
        rows.append(table + [-1] * (width - len(table)))
        lens.append(lengths[s] + m)
    return rows, lens, slots, positions, owner


def attention(q, k_codes, v_codes, k_scale, v_scale, tables, kv_len, cu, *, scale, window=0, softcap=0.0):
    """(out, lse, A, X): A = sum p |v|, X = max over the seen keys of scale * sum |q| |k|."""
    t, heads, d = q.shape
    pages, kvh, page, _ = k_codes.shape
    out = torch.zeros(t, heads, d, dtype=torch.float64, device=q.device)
    spread = torch.zeros_like(out)
    lse = torch.full((t, heads), -math.inf, dtype=torch.float64, device=q.device)
    reach = torch.zeros_like(lse)
    for r, n in enumerate(kv_len.tolist()):
        a, b = int(cu[r]), int(cu[r + 1])
        if n <= 0 or b <= a:
            continue
        held = tables[r, : -(-n // page)].long()
        k = (k_codes[held].double() * k_scale[held].double()[..., None, None]).transpose(0, 1).reshape(kvh, -1, d)[:, :n]
        v = (v_codes[held].double() * v_scale[held].double()[..., None, None]).transpose(0, 1).reshape(kvh, -1, d)[:, :n]
        for i in range(a, b):
            pos = n - (b - a) + i - a
            low = max(0, pos - window + 1) if window else 0
            if pos < low:
                continue
            qi = q[i].double().view(kvh, heads // kvh, d)
            x = scale * torch.einsum("hgd,hkd->hgk", qi, k[:, low:pos + 1])
            big = scale * torch.einsum("hgd,hkd->hgk", qi.abs(), k[:, low:pos + 1].abs())
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            lse[i] = torch.logsumexp(x, 2).view(heads)
            p = torch.softmax(x, 2)
            out[i] = torch.einsum("hgk,hkd->hgd", p, v[:, low:pos + 1]).reshape(heads, d)
            spread[i] = torch.einsum("hgk,hkd->hgd", p, v[:, low:pos + 1].abs()).reshape(heads, d)
            reach[i] = big.amax(2).view(heads)
    return out, lse, spread, reach


def rms_norm(x, residual, weight, *, eps):
    """(h, y)."""
    h = x.double() + (0.0 if residual is None else residual.double())
    return h, h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * weight.double()


def w4_product(x, x_scale, codes, scales):
    """(out, sum |w| |x|)."""
    out, half = codes.shape
    k = 2 * half
    n = torch.empty(out, k, dtype=torch.float64, device=codes.device)
    n[:, 0::2], n[:, 1::2] = (codes % 16).double() - 8, (codes // 16).double() - 8
    w = n * scales.double().repeat_interleave(k // scales.shape[1], 1)
    x = x.double()
    if x_scale is not None:
        x = x * x_scale.double().repeat_interleave(k // x_scale.shape[1], 1)
    return x @ w.t(), x.abs() @ w.abs().t()


def head_norm_rotary(x, weight, positions, frequencies, *, rotary, pairs, eps, norm=True):
    """x [tokens, heads, dim] normed by head and rotated; frequencies: radians a position, as Python floats."""
    y = x.double()
    if norm:
        y = y / torch.sqrt((y * y).mean(2, keepdim=True) + eps)
        y = y if weight is None else y * weight.double()
    angle = torch.tensor([[math.remainder(p * f, 2 * math.pi) for f in frequencies] for p in positions.tolist()],
                         dtype=torch.float64, device=x.device).view(-1, 1, rotary // 2)
    a, b = (y[..., : rotary // 2], y[..., rotary // 2:rotary]) if pairs == "halves" else (y[..., 0:rotary:2], y[..., 1:rotary:2])
    turned = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
    turned = torch.cat(turned, 2) if pairs == "halves" else torch.stack(turned, 3).flatten(2)
    return torch.cat([turned, y[..., rotary:]], 2)


def sample(logits, u, *, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob) of one row of logits, over Python numbers."""
    x = [v if v == v else -math.inf for v in logits.double().tolist()]
    order = sorted((i for i in range(len(x)) if x[i] > -math.inf), key=lambda i: (-x[i], i))
    if not order:
        return -1, -math.inf
    if temperature == 0.0:
        return order[0], 0.0
    top = x[order[0]]
    mass = {i: 1 << 45 if x[i] == top else round(2.0 ** 45 * math.exp((x[i] - top) / temperature)) for i in order}
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1.0:
        limit, before, kept = max(1, math.ceil(top_p * float(sum(mass[i] for i in order)))), 0, []
        for i in order:
            if before >= limit:
                break
            kept.append(i)
            before += mass[i]
        order = kept
    order = sorted(i for i in order if mass[i] >= math.ceil(min_p * 2.0 ** 45) and mass[i] > 0)
    total = sum(mass[i] for i in order)
    target, upto = min(total - 1, math.floor(u * float(total))), 0
    for i in order:
        upto += mass[i]
        if upto > target:
            return i, math.log(mass[i] / total)


def gated(x, x_scale, codes, scales, *, activation):
    """(out, bound on out's error for products off by e * sum |w||x| each, as a function of e)."""
    y, reach = w4_product(x, x_scale, codes, scales)
    g, u = y.chunk(2, 1)
    dg, du = reach.chunk(2, 1)
    z = g if activation == "silu" else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    act = g * torch.sigmoid(z)
    # neither activation is steeper than 1.13 anywhere, nor larger than its argument
    return act * u, lambda e: e * (1.13 * dg * u.abs() + act.abs() * du + 1.13 * e * dg * du)
