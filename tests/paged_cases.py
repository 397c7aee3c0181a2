"""Inputs of the tests of paged caches: sequences of given lengths in pages in any order, the pages' unused rows full of what must not be read."""
from __future__ import annotations

from types import SimpleNamespace

import torch

BF16 = torch.bfloat16
NAN = float("nan")


def table_of(g, totals, page, spare=2, entries=None):
    """Page numbers [B, entries] of sequences of these lengths, in any order; entries behind a sequence's last page name no page."""
    need = [-(-t // page) for t in totals]
    order = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    table = torch.full((len(totals), max([1, *need]) if entries is None else entries), -7, dtype=torch.int32)
    first = 0
    for b, n in enumerate(need):
        table[b, :n] = order[first:first + n]
        first += n
    return table, len(order)


def attention_case(new, totals, Hq, Hkv, D, page, device, seed=0, packed=True, spare_rows=0, rubbish=NAN, entries=None):
    """Queries of sequences with `new` new tokens of `totals` in all, their cache and table on the device.  The cache's rows that belong to no
    token hold `rubbish`.  packed: rows one behind the other (with `starts`, and spare_rows behind the last), else [B, T, Hq, D]."""
    g = torch.Generator().manual_seed(seed)
    table, pages = table_of(g, totals, page, entries=entries)
    caches = []
    for _ in range(2):
        c = torch.full((pages, page, Hkv, D), rubbish, dtype=BF16)
        for b, t in enumerate(totals):
            at = torch.arange(t)
            c[table[b].long()[at // page], at % page] = torch.randn(t, Hkv, D, generator=g).to(BF16)
        caches.append(c.to(device))
    rows = sum(new)
    q = torch.randn(rows + spare_rows, Hq, D, generator=g).to(BF16).to(device)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    if not packed:
        assert len(set(new)) == 1 and spare_rows == 0
    return SimpleNamespace(q=q if packed else q.view(len(new), new[0], Hq, D), rows=q, k=caches[0], v=caches[1], table=table.to(device), starts=starts,
                           seq_lens=torch.tensor(totals, dtype=torch.int32, device=device),
                           starts_arg=torch.tensor(starts, dtype=torch.int32, device=device) if packed else None)
