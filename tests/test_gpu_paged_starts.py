"""Packed rows that are no partition: `starts` that do not ascend name the same rows for many sequences.  No call is to be made so, and nothing may
be written out of place for it."""
import pytest
import torch

from paged_cases import BF16

pytestmark = pytest.mark.gpu


def test_rows_named_more_often_than_can_be_counted(ext, device):
    # 1000 times the same 8192 rows behind a million keys (all in one page): 1000 x 8 heads x 128 units x 2 x 8192 columns are more than 32 bits hold
    B, rows, page, keys = 2000, 8192, 16384, 1 << 20
    k = torch.zeros(1, page, 8, 64, dtype=BF16, device=device)
    q = torch.zeros(rows, 32, 64, dtype=BF16, device=device)
    table = torch.zeros(1, keys // page, dtype=torch.int32, device=device).expand(B, -1)
    starts = torch.tensor([0, rows] * (B // 2) + [0], dtype=torch.int32, device=device)
    assert 1000 * 8 * 128 * (2 * 8192 + 1) > 2 ** 32
    out = torch.full_like(q, 7.0)
    ext.paged_attention(q, k, k, table, torch.full((B,), keys, dtype=torch.int32, device=device), starts=starts, out=out)
    assert bool((out == 7.0).all())
    # the rows of a call that does name each once
    good = torch.tensor([0, 5, rows] + [rows] * (B - 2), dtype=torch.int32, device=device)
    ext.paged_attention(q, k, k, table, torch.full((B,), 300, dtype=torch.int32, device=device), starts=good, out=out)
    assert bool((out == 0.0).all())
