"""Norms of query and key heads, rotation and the append to a paged cache in one pass, against the formula in 64 bits.

Tolerance: one rounding to bf16 (2^-8 of the result) and about ten roundings in 32 bits (2^-24 of the pair's size each): 2^-20 of that."""
import pytest
import torch

from oracle import paged
from oracle.rope import freqs_cis_reference
from oracle import inputs
from paged_cases import BF16, table_of

pytestmark = pytest.mark.gpu


def make(device, new, positions, Hq, Hkv, D, page, norms, seed=0, spare_rows=0, entries=None, freq_rows=None):
    g = torch.Generator().manual_seed(seed)
    totals = [n + p for n, p in zip(new, positions)]
    table, pages = table_of(g, totals, page, entries=entries)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    rows = starts[-1] + spare_rows
    c = dict(qkv=torch.randn(rows, (Hq + 2 * Hkv) * D, generator=g).to(BF16), freq=freqs_cis_reference(D, freq_rows or max(totals), **inputs.ROPE_CONFIG4).contiguous(),
             cache_k=torch.full((pages, page, Hkv, D), 3.0, dtype=BF16), cache_v=torch.full((pages, page, Hkv, D), 5.0, dtype=BF16), page_table=table,
             positions=torch.tensor(positions, dtype=torch.int32))
    if norms:
        c.update(q_norm=(1 + 0.2 * torch.randn(D, generator=g)).to(BF16), k_norm=(1 + 0.2 * torch.randn(D, generator=g)).to(BF16))
    c = {k: v.to(device) for k, v in c.items()}
    return c, starts, torch.tensor(starts, dtype=torch.int32, device=device)


def check(c, starts, Hq, Hkv, q, q_before, eps=1e-5):
    names = {k: v for k, v in c.items() if k not in ("positions", "page_table")}
    want = paged.append(names["qkv"].reshape(-1, names["qkv"].shape[-1]), names["freq"], c["cache_k"], c["cache_v"], c["page_table"].cpu(), c["positions"].cpu(), starts, Hq, Hkv,
                        names.get("q_norm"), names.get("k_norm"), eps)
    D = c["cache_k"].shape[-1]
    for name, got, before in (("q", q.reshape(-1, Hq, D), q_before), ("k", c["cache_k"].reshape(-1, Hkv, D), 3.0), ("v", c["cache_v"].reshape(-1, Hkv, D), 5.0)):
        at, value, size = want[name]
        off = (got[at].double() - value).abs()
        assert bool((off <= value.abs() * 2 ** -8 + size * 2 ** -20 + 1e-38).all()), name
        other = torch.ones(got.shape[0], dtype=torch.bool, device=got.device)
        other[at] = False
        assert bool((got[other] == before).all()), f"{name}: rows of no token are left as they were"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (3, 1), (24, 8)])
@pytest.mark.parametrize("norms", [False, True])
def test_packed_rows(ext, device, D, Hq, Hkv, norms):
    c, starts, dev_starts = make(device, [3, 0, 1, 70, 1, 16], [0, 9, 31, 5, 200, 16], Hq, Hkv, D, 16, norms, seed=D + Hq, spare_rows=3)
    out = torch.full((starts[-1] + 3, Hq, D), 9.0, dtype=BF16, device=device)
    q = ext.rot_embed_paged_kv_cache(**c, n_head=Hq, n_kv_head=Hkv, starts=dev_starts, out=out)
    assert q.data_ptr() == out.data_ptr()
    check(c, starts, Hq, Hkv, q, 9.0)


@pytest.mark.parametrize("D", [8, 40, 72, 96, 200, 256])
@pytest.mark.parametrize("norms", [False, True])
def test_other_head_sizes_and_pages(ext, device, D, norms):
    c, starts, dev_starts = make(device, [5, 9], [2, 30], 5, 2, D, 7, norms, seed=D)
    check(c, starts, 5, 2, ext.rot_embed_paged_kv_cache(**c, n_head=5, n_kv_head=2, starts=dev_starts, eps=1e-3), 9.0, eps=1e-3)


@pytest.mark.parametrize("T", [1, 5])
def test_batches_of_equal_chunks_and_strides(ext, device, T):
    B, Hq, Hkv, D = 6, 8, 2, 64
    c, starts, _ = make(device, [T] * B, [7 * b for b in range(B)], Hq, Hkv, D, 32, True, seed=T)
    rows = c["qkv"]
    wide = torch.zeros(T, B, rows.shape[1] + 16, dtype=BF16, device=device)
    wide[..., 8:-8] = rows.view(B, T, -1).transpose(0, 1)
    both = torch.stack([c["cache_k"], c["cache_v"]], dim=1)
    c["cache_k"], c["cache_v"] = both[:, 0], both[:, 1]
    q = ext.rot_embed_paged_kv_cache(**{**c, "qkv": wide[..., 8:-8].transpose(0, 1)}, n_head=Hq, n_kv_head=Hkv)
    assert q.shape == (B, T, Hq, D)
    check(c, starts, Hq, Hkv, q, 9.0)


def test_without_norms_the_bits_of_the_dense_cache(ext, device):
    B, T, Hq, Hkv, D, page = 4, 3, 8, 2, 128, 16
    c, starts, _ = make(device, [T] * B, [0, 5, 14, 40], Hq, Hkv, D, page, False, seed=2)
    qkv = c["qkv"].view(B, T, -1)
    length = c["page_table"].shape[1] * page
    ck, cv = (torch.zeros(B, length, Hkv, D, dtype=BF16, device=device) for _ in range(2))
    want = ext.rot_embed_kv_cache(qkv, c["freq"], ck, cv, 0, Hq, Hkv, positions=c["positions"])
    got = ext.rot_embed_paged_kv_cache(**{**c, "qkv": qkv}, n_head=Hq, n_kv_head=Hkv)
    assert torch.equal(got, want)
    for b, p in enumerate((0, 5, 14, 40)):
        at = torch.arange(p, p + T, device=device)
        pages = c["page_table"][b].long()[at // page]
        assert torch.equal(c["cache_k"][pages, at % page], ck[b, p:p + T]) and torch.equal(c["cache_v"][pages, at % page], cv[b, p:p + T])


def test_tokens_without_a_place_are_skipped(ext, device):
    # before the table, behind the rotary table, behind the pages, on a page that is not there
    c, starts, dev_starts = make(device, [4, 4, 4, 4], [10, 20, 30, 40], 4, 2, 64, 16, True, seed=1, entries=4)
    c["positions"].copy_(torch.tensor([-2, 41, 62, 15], dtype=torch.int32))
    c["page_table"][3, 1] = 10 ** 6
    c["page_table"][2] = c["page_table"][2, 0]
    out = torch.full((16, 4, 64), 9.0, dtype=BF16, device=device)
    ext.rot_embed_paged_kv_cache(**c, n_head=4, n_kv_head=2, starts=dev_starts, out=out)
    check(c, starts, 4, 2, out, 9.0)


def test_many_sequences_and_captured_steps(ext, device):
    B = 700
    c, starts, dev_starts = make(device, [1 + b % 3 for b in range(B)], [b % 50 for b in range(B)], 4, 1, 64, 16, True, seed=3)
    out = torch.full((starts[-1], 4, 64), 9.0, dtype=BF16, device=device)
    ext.rot_embed_paged_kv_cache(**c, n_head=4, n_kv_head=1, starts=dev_starts, out=out)
    check(c, starts, 4, 1, out, 9.0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q = ext.rot_embed_paged_kv_cache(**c, n_head=4, n_kv_head=1, starts=dev_starts)
    c["positions"] -= 1          # (those at 0 fall out)
    c["cache_k"].fill_(3.0), c["cache_v"].fill_(5.0)
    q.fill_(9.0)
    g.replay()
    check(c, starts, 4, 1, q, 9.0)


def test_refusals(ext, device):
    c, _, dev_starts = make(device, [2, 2], [0, 3], 4, 2, 64, 16, True)
    good = dict(c, n_head=4, n_kv_head=2, starts=dev_starts)
    ext.rot_embed_paged_kv_cache(**good)
    bad = [
        (dict(qkv=c["qkv"].float()), "bfloat16"), (dict(qkv=c["qkv"][None]), "packed|with starts"), (dict(n_head=5), "head counts"), (dict(n_head=2, n_kv_head=3), "n_kv_head, D"),
        (dict(freq=c["freq"].double()), "float32"), (dict(freq=c["freq"][:, :32]), "whole float32"), (dict(q_norm=None), "go together"),
        (dict(k_norm=c["k_norm"][:32]), r"\[D\]"), (dict(positions=c["positions"].long()), "int32"), (dict(page_table=c["page_table"][:1]), r"\[B\]"),
        (dict(starts=dev_starts[:2]), r"\[B \+ 1\]"), (dict(cache_v=c["cache_v"].transpose(0, 1)), "equal layout"), (dict(out=torch.zeros(4, 4, 32, dtype=BF16, device=device)), "n_head, D"),
        (dict(qkv=torch.zeros(4, 8 * 64 + 4, dtype=BF16, device=device)[:, 4:]), "16 bytes"),
    ]
    for change, words in bad:
        with pytest.raises(RuntimeError, match=words):
            ext.rot_embed_paged_kv_cache(**{**good, **change})
    with pytest.raises(RuntimeError, match="multiple of 8"):
        ext.rot_embed_paged_kv_cache(torch.zeros(1, 1, 4 * 12, dtype=BF16, device=device), torch.zeros(4, 12, device=device), torch.zeros(2, 16, 1, 12, dtype=BF16, device=device),
                                     torch.zeros(2, 16, 1, 12, dtype=BF16, device=device), torch.zeros(1, 1, dtype=torch.int32, device=device),
                                     torch.zeros(1, dtype=torch.int32, device=device), 2, 1)
