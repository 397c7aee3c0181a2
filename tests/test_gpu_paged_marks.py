"""Attention of chunks over a paged cache: values that are no numbers, taken out of some of the many short segments that a block goes through.  The marks of
its ring of segments are used again and again: each belongs to its own segment."""
import pytest
import torch

from paged_cases import NAN, attention_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [9, 40])
def test_marks_of_segments_go_with_their_segments(ext, device, D, new):
    # 500 sequences x 8 heads of one unit each: 27 units a block.  Every third sequence's last value row holds a NaN and an infinity for two of its heads: the
    # tokens before the last do not see them, the last one does, and all other sequences have what they had
    B, Hkv, total = 500, 8, 70
    clean = attention_case([new] * B, [total] * B, 16, Hkv, D, 16, device, seed=new + D)
    want = ext.paged_attention(clean.q, clean.k, clean.v, clean.table, clean.seq_lens, starts=clean.starts_arg)
    odd = torch.arange(0, B, 3, device=device)
    pages, at = clean.table[odd, (total - 1) // 16].long(), (total - 1) % 16
    values = clean.v.clone()
    values[pages, at, 1, 3], values[pages, at, 6, D - 1] = NAN, float("inf")
    want = want.view(B, new, Hkv, 2, D)
    mine = torch.zeros_like(want, dtype=torch.bool)
    mine[odd, new - 1, 1, :, 3] = mine[odd, new - 1, 6, :, D - 1] = True
    for _ in range(3):
        got = ext.paged_attention(clean.q, clean.k, values, clean.table, clean.seq_lens, starts=clean.starts_arg).view_as(want)
        assert torch.equal(got[~mine], want[~mine])
        assert torch.isnan(got[odd, new - 1, 1, :, 3]).all() and (got[odd, new - 1, 6, :, D - 1] == float("inf")).all()
