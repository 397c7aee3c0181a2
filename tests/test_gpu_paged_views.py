"""Views that the calls on paged caches take, an axis of one entry at any stride, and one that they refuse."""
import pytest
import torch

from paged_cases import BF16

pytestmark = pytest.mark.gpu
ODD = 13      # a stride that no 16-byte vector has


def odd(t):
    """t with its axes of one entry at an odd stride."""
    return t.as_strided(t.shape, [ODD if n == 1 else s for n, s in zip(t.shape, t.stride())])


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv", [(1, 1, 1), (1, 8, 2), (40, 1, 1), (40, 8, 2)])
def test_axes_of_one_entry(ext, device, packed, T, Hq, Hkv):
    D, page = 64, 64
    g = torch.Generator().manual_seed(T + Hq)
    r = lambda *s: torch.randn(*s, generator=g).to(BF16).to(device)  # noqa: E731
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    k, v, freq = r(1, page, Hkv, D), r(1, page, Hkv, D), torch.randn(page, D, generator=g).to(device)
    qkv = r(1, T, (Hq + 2 * Hkv) * D)
    table, first, length, starts = torch.zeros(1, 1, dtype=torch.int32, device=device), ints(7), ints(7 + T), ints(0, T) if packed else None
    rows = (lambda t: t[0]) if packed else (lambda t: t)
    plain, views = (k.clone(), v.clone()), (odd(k.clone()), odd(v.clone()))
    want = ext.rot_embed_paged_kv_cache(rows(qkv), freq, *plain, table, first, Hq, Hkv, starts=starts)
    got = ext.rot_embed_paged_kv_cache(odd(rows(qkv)), freq, *views, table, first, Hq, Hkv, starts=starts)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(plain, views))
    y = ext.paged_attention(want, *plain, table, length, starts=starts)
    out = torch.zeros_like(y)
    ext.paged_attention(odd(want), *views, table, length, starts=starts, out=odd(out))
    assert torch.equal(out, y)


def test_more_tokens_than_are_counted_in_32_bits(ext, device):
    # (a broadcast token, which needs no memory; 2^32 + 1 is 1 in 32 bits)
    k = torch.zeros(1, 16, 1, 8, dtype=BF16, device=device)
    many = torch.zeros(1, 1, 24, dtype=BF16, device=device).expand(1, 2 ** 32 + 1, 24)
    with pytest.raises(RuntimeError, match="too large"):
        ext.rot_embed_paged_kv_cache(many, torch.zeros(16, 8, device=device), k, k.clone(), torch.zeros(1, 1, dtype=torch.int32, device=device),
                                     torch.zeros(1, dtype=torch.int32, device=device), 1, 1)
