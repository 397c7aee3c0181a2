"""Paged caches and adapters from their formulas in 64 bits, token by token and sequence by sequence.

A paged cache is [pages, page_size, heads, D]; token p of sequence b lies in row p % page_size of page table[b, p // page_size].
New tokens lie one behind the other: sequence b has rows [starts[b], starts[b + 1])."""
from __future__ import annotations

import torch

F64 = torch.float64


def uniform_starts(B: int, T: int) -> list:
    return [b * T for b in range(B + 1)]


def rows_of(cache, table_row, n: int):
    """The first n tokens of a sequence [n, heads, D]; pages that are not there are zeros."""
    pages, page = cache.shape[:2]
    at = torch.arange(n, device=cache.device)
    number = table_row.to(cache.device).long()[at // page]
    there = (number >= 0) & (number < pages)
    return torch.where(there[:, None, None], cache[number.clamp(0, max(pages - 1, 0)), at % page], torch.zeros((), dtype=cache.dtype, device=cache.device))


def rotated(x, turn):
    """x [n, heads, D] of interleaved pairs by turn [n, D] = (cos, sin) of every pair; and the size of each entry's pair."""
    n, H, D = x.shape
    x = x.reshape(n, H, D // 2, 2)
    c, s = turn.reshape(n, 1, D // 2, 2).unbind(-1)
    out = torch.stack([x[..., 0] * c - x[..., 1] * s, x[..., 0] * s + x[..., 1] * c], dim=-1)
    size = x.abs().sum(-1, keepdim=True).expand_as(x)
    return out.reshape(n, H, D), size.reshape(n, H, D)


def append(qkv, freq, cache_k, cache_v, table, positions, starts, Hq, Hkv, q_norm=None, k_norm=None, eps=1e-5):
    """qkv [rows, (Hq + 2 Hkv) D].  Returns per entry written {name: (flat row numbers, values in 64 bits, pair sizes)} for "q", "k", "v":
    rows of the queries, and rows of the caches as [pages * page_size]."""
    D = qkv.shape[-1] // (Hq + 2 * Hkv)
    pages, page = cache_k.shape[:2]
    x = qkv.to(F64).reshape(qkv.shape[0], Hq + 2 * Hkv, D)
    rows, at, slot = [], [], []
    for b in range(len(starts) - 1):
        for r in range(starts[b], starts[b + 1]):
            p = int(positions[b]) + r - starts[b]
            if not 0 <= p < freq.shape[0] or p // page >= table.shape[1]:
                continue
            number = int(table[b, p // page])
            if 0 <= number < pages:
                rows.append(r), at.append(p), slot.append(number * page + p % page)
    rows, at, slot = (torch.tensor(v, dtype=torch.long, device=qkv.device) for v in (rows, at, slot))
    q, k, v = x[rows].split([Hq, Hkv, Hkv], dim=1)
    if q_norm is not None:
        q = q / (q.square().mean(-1, keepdim=True) + eps).sqrt() * q_norm.to(F64)
        k = k / (k.square().mean(-1, keepdim=True) + eps).sqrt() * k_norm.to(F64)
    turn = freq.to(F64)[at]
    return {"q": (rows, *rotated(q, turn)), "k": (slot, *rotated(k, turn)), "v": (slot, v, v.abs())}


def attention(q, cache_k, cache_v, table, seq_lens, starts, scale=None):
    """q [rows, Hq, D].  Returns the results in 64 bits, their sums of p |v|, and which rows belong to a sequence."""
    rows, Hq, D = q.shape
    Hkv = cache_k.shape[2]
    scale = D ** -0.5 if not scale else scale
    out = torch.zeros(rows, Hq, D, dtype=F64, device=q.device)
    size, mine = torch.zeros_like(out), torch.zeros(rows, dtype=torch.bool, device=q.device)
    for b in range(len(starts) - 1):
        r0, r1 = starts[b], starts[b + 1]
        n, length = r1 - r0, min(max(int(seq_lens[b]), 0), table.shape[1] * cache_k.shape[1])
        if n == 0:
            continue
        mine[r0:r1] = True
        k, v = (rows_of(c, table[b], length).to(F64).repeat_interleave(Hq // Hkv, dim=1) for c in (cache_k, cache_v))
        for t in range(n):       # (a token's own keys only: what it must not see does not enter the sums)
            seen = length - n + t + 1
            if seen <= 0:
                continue
            s = torch.einsum("hd,jhd->hj", q[r0 + t].to(F64), k[:seen]) * scale
            p = torch.softmax(s, dim=-1)
            out[r0 + t] = torch.einsum("hj,jhd->hd", p, v[:seen])
            size[r0 + t] = torch.einsum("hj,jhd->hd", p, v[:seen].abs())
    return out, size, mine


def adapter_linear(x, w, a, b, index, scales=None):
    """x [rows, K].  Returns the results in 64 bits, the sums of |x w|, and of |s| |z| |b| with |z| the sums of |x a|."""
    x64, w64 = x.to(F64), w.to(F64)
    y, size = x64 @ w64.T, x64.abs() @ w64.abs().T
    low = torch.zeros_like(y)
    for i in sorted(set(index.tolist())):
        if 0 <= i < a.shape[0]:
            at = (index == i).nonzero().view(-1).to(x.device)
            s = 1.0 if scales is None else float(scales[i])
            a64, b64 = a[i].to(F64), b[i].to(F64)
            y[at] += s * (x64[at] @ a64.T) @ b64.T
            low[at] = abs(s) * (x64[at].abs() @ a64.abs().T) @ b64.abs().T
    return y, size, low
