"""Attention of new tokens over a paged cache against the formula in 64 bits.

Tolerance: the result is rounded to bf16 (2^-8 of its size), and so are the weights p of the values (2^-8 of the sum of p |v|, `size`); what is
left are scores in 32 bits, whose error of D 2^-24 |q| |k| scale (below 2^-13 for normal inputs of these sizes) moves a weight by as much."""
import pytest
import torch

from oracle import paged
from paged_cases import BF16, NAN, attention_case

pytestmark = pytest.mark.gpu


def check(got, case, scale=None):
    want, size, mine = paged.attention(case.rows, case.k, case.v, case.table, case.seq_lens, case.starts, scale)
    got = got.reshape(want.shape).double()
    off = (got - want).abs()[mine]
    bound = (want.abs() * 2 ** -8 + size * (2 ** -8 + 2 ** -12) + 1e-30)[mine]
    assert torch.isfinite(got[mine]).all()
    assert bool((off <= bound).all()), f"{(off / bound).max().item():.3g} of the bound"


def run(ext, case, **kw):
    return ext.paged_attention(case.q, case.k, case.v, case.table, case.seq_lens, starts=case.starts_arg, **kw)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (6, 2), (16, 1), (10, 2), (7, 1)])
@pytest.mark.parametrize("page", [16, 48])
def test_single_tokens(ext, device, D, Hq, Hkv, page):
    totals = [1, 2, 15, 16, 17, 33, 129, 500, 1027]
    case = attention_case([1] * len(totals), totals, Hq, Hkv, D, page, device, seed=Hq + D + page, packed=False)
    check(run(ext, case), case)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (8, 2), (12, 4), (16, 1), (5, 1)])
@pytest.mark.parametrize("page", [16, 64, 96, 256])
def test_packed_rows_of_every_length(ext, device, D, Hq, Hkv, page):
    new = [3, 0, 1, 64, 130, 1, 2, 17, 300, 1]
    totals = [3, 5, 400, 64, 333, 1, 130, 145, 777, 2049]
    case = attention_case(new, totals, Hq, Hkv, D, page, device, seed=page + D + Hq, spare_rows=5)
    out = torch.full_like(case.q, 7.0)
    assert run(ext, case, out=out) is not None
    check(out, case)
    assert bool((out[sum(new):] == 7.0).all()), "rows behind the last sequence are left as they were"


@pytest.mark.parametrize("T", [1, 2, 4, 5, 16, 31, 33, 64, 127, 128, 129, 257])
@pytest.mark.parametrize("D", [64, 128])
def test_uniform_chunks(ext, device, T, D):
    case = attention_case([T, T, T], [T, T + 200, T + 1001], 8, 2, D, 32, device, seed=T, packed=False)
    check(run(ext, case), case)


@pytest.mark.parametrize("T,total", [(512, 4500), (1, 30011), (3, 30011), (700, 700)])
def test_long_sequences(ext, device, T, total):
    case = attention_case([T], [total], 8, 2, 128, 16, device, seed=T, packed=False)
    check(run(ext, case), case)


def test_many_short_sequences_beside_one_long(ext, device):
    new, totals = [1] * 300 + [200], [1 + 7 * i % 90 for i in range(300)] + [9000]
    case = attention_case(new, totals, 8, 2, 64, 16, device, seed=5)
    check(run(ext, case), case)


def test_more_sequences_than_a_launch_takes(ext, device):
    # 2048 sequences a launch: one token each, and packed rows with a chunk on either side of the border
    totals = [1 + 5 * i % 37 for i in range(2500)]
    case = attention_case([1] * 2500, totals, 4, 2, 64, 16, device, seed=1, packed=False)
    check(run(ext, case), case)
    new = [1] * 2040 + [20, 3, 0, 70, 1, 1, 9, 2, 33, 1] + [1] * 30
    case = attention_case(new, [n + i % 41 for i, n in enumerate(new)], 4, 2, 64, 16, device, seed=2)
    check(run(ext, case), case)


@pytest.mark.parametrize("new", [1, 70])
def test_queries_that_are_broadcast(ext, device, new):
    case = attention_case([new] * 3, [100, 200, 300], 8, 2, 64, 16, device, seed=new, packed=False)
    one = case.q[:1, :, :1]
    got = ext.paged_attention(one.expand(3, new, 8, 64), case.k, case.v, case.table, case.seq_lens)
    case.rows = one.expand(3, new, 8, 64).reshape(-1, 8, 64).contiguous()
    check(got, case)


@pytest.mark.parametrize("D", [64, 128])
def test_sequences_that_share_pages_and_results_in_the_place_of_queries(ext, device, D):
    case = attention_case([1, 90, 3, 1], [700, 690, 803, 640], 8, 2, D, 16, device, seed=D)
    case.table[1:, :30] = case.table[0, :30]          # 480 tokens in common
    apart = run(ext, case)
    check(apart, case)
    case.rows = case.q.clone()
    assert run(ext, case, out=case.q) is not None
    assert torch.equal(case.q, apart)


def test_lengths_that_leave_tokens_without_keys(ext, device):
    # fewer tokens cached than are new: the first ones see nothing; a length of zero; one beyond the table's row is clamped
    case = attention_case([5, 40, 3, 1, 300], [64, 64, 64, 64, 320], 8, 2, 128, 16, device, seed=9)
    case.seq_lens = torch.tensor([2, 17, 0, -3, 100], dtype=torch.int32, device=device)
    out = run(ext, case)
    check(out, case)
    assert bool((out[:3] == 0).all()) and bool((out[5:28] == 0).all()) and bool((out[45:49] == 0).all()) and bool((out[49:249] == 0).all())
    one = attention_case([1, 1], [64, 64], 8, 2, 64, 16, device, seed=10, packed=False)
    one.seq_lens = torch.tensor([0, 10 ** 6], dtype=torch.int32, device=device)
    out = run(ext, one)
    check(out, one)
    assert bool((out[0] == 0).all())


@pytest.mark.parametrize("new,total", [(4, 40), (2, 130), (3, 16), (64, 300), (200, 200), (130, 1000)])
@pytest.mark.parametrize("D", [64, 128])
def test_values_that_are_no_numbers_stay_with_the_tokens_that_see_them(ext, device, D, new, total):
    # the last new tokens' values hold a NaN and infinities, their keys too: earlier tokens do not see them
    case = attention_case([new], [total], 8, 2, D, 16, device, seed=new + D)
    page = int(case.table[0, (total - 1) // 16])
    at = (total - 1) % 16
    case.v[page, at, 0, 3], case.v[page, at, 1, D - 1] = NAN, float("inf")
    case.v[page, at, 1, 5] = float("-inf")
    clean = attention_case([new], [total], 8, 2, D, 16, device, seed=new + D)
    got = run(ext, case)
    want = run(ext, clean)
    assert torch.equal(got[:new - 1], want[:new - 1])
    last, same = got[new - 1], want[new - 1]
    assert torch.isnan(last[:4, 3]).all() and (last[4:, D - 1] == float("inf")).all() and (last[4:, 5] == float("-inf")).all()
    rest = torch.ones(8, D, dtype=torch.bool, device=device)
    rest[:4, 3] = rest[4:, D - 1] = rest[4:, 5] = False
    assert torch.equal(last[rest], same[rest])
    # a key that is no number: the tokens that see it have no result, the others theirs
    clean.k[page, at, 0, 0] = NAN
    got = run(ext, clean)
    assert torch.equal(got[:new - 1], want[:new - 1]) and torch.isnan(got[new - 1, :4]).all() and torch.equal(got[new - 1, 4:], want[new - 1, 4:])


@pytest.mark.parametrize("new", [1, 3, 90])
def test_pages_that_are_not_there_count_as_zeros(ext, device, new):
    case = attention_case([new, new], [200, 200], 8, 2, 64, 16, device, seed=new)
    case.table[0, 3], case.table[1, 0], case.table[1, 2] = -1, 2 ** 31 - 1, case.k.shape[0]
    check(run(ext, case), case)


@pytest.mark.parametrize("new", [1, 100])
def test_strided_inputs_and_outputs(ext, device, new):
    # caches that are two halves of one tensor, heads of a wider query tensor, a table of wider rows, an output of another layout
    case = attention_case([new] * 3, [300] * 3, 8, 2, 128, 32, device, seed=4, packed=False)
    both = torch.stack([case.k, case.v], dim=1)
    wide = torch.zeros(3, new, 13, 128, dtype=BF16, device=device)
    wide[:, :, 2:10] = case.q
    table = torch.full((3, 40), -1, dtype=torch.int32, device=device)
    table[:, 5:5 + case.table.shape[1]] = case.table
    out = torch.empty(8, new, 3, 128, dtype=BF16, device=device).permute(2, 1, 0, 3)
    got = ext.paged_attention(wide[:, :, 2:10], both[:, 0], both[:, 1], table[:, 5:5 + case.table.shape[1]], case.seq_lens, out=out)
    assert got.data_ptr() == out.data_ptr()
    check(out, case)


def test_scale_and_large_scores(ext, device):
    for new in (1, 70):
        case = attention_case([new], [500], 4, 2, 64, 16, device, seed=3)
        case.q *= 8
        case.rows = case.q
        check(run(ext, case, scale=0.25), case, scale=0.25)


def test_pages_behind_two_gigabytes(ext, device):
    # offsets of the cache beyond 32 bits: 40 pages spread over 8 GB
    page, Hkv, D = 256, 8, 128
    pages = 8400   # x 256 x 8 x 128 = 2.2e9 elements
    k, v = (torch.empty(pages, page, Hkv, D, dtype=BF16, device=device) for _ in range(2))
    table = torch.arange(pages - 1, pages - 21, -1, dtype=torch.int32, device=device).view(2, 10)
    k[table.view(-1).long()] = torch.randn(20, page, Hkv, D, device=device).to(BF16)
    v[table.view(-1).long()] = torch.randn(20, page, Hkv, D, device=device).to(BF16)
    for new in (1, 65):
        q = torch.randn(2, new, 16, D, device=device).to(BF16)
        lens = torch.tensor([2500, 1300], dtype=torch.int32, device=device)
        got = ext.paged_attention(q, k, v, table, lens)
        want, size, _ = paged.attention(q.flatten(0, 1), k, v, table, lens, paged.uniform_starts(2, new))
        assert bool(((got.flatten(0, 1).double() - want).abs() <= want.abs() * 2 ** -8 + size * (2 ** -8 + 2 ** -12)).all())


def test_same_bits_every_time_and_on_another_stream(ext, device):
    case = attention_case([1, 40, 1, 2], [3000, 900, 77, 5000], 8, 2, 128, 16, device, seed=1)
    first = run(ext, case)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [run(ext, case) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    again += [run(ext, case) for _ in range(3)]
    assert all(torch.equal(first, a) for a in again)


def test_two_graphs_at_once_and_lengths_that_change_between_replays(ext, device):
    cases = [attention_case([1] * 5, [900, 10, 33, 2000, 1], 8, 2, 64, 16, device, seed=s, packed=False) for s in (1, 2)]
    run(ext, cases[0])
    graphs, outs, side = [], [], torch.cuda.Stream()
    for case in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(ext, case))
        graphs.append(g)
    for shift in (0, 5):
        for case in cases:
            case.seq_lens.copy_(torch.tensor([900 - 7 * shift, 10 - shift, 33, 2000 - 100 * shift, 1], dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(20):
            graphs[0].replay()
            with torch.cuda.stream(side):
                graphs[1].replay()
        torch.cuda.synchronize()
        for case, out in zip(cases, outs):
            check(out, case)


def test_scratch_that_holds_no_numbers(ext, device):
    case = attention_case([1, 40, 1, 2, 300], [3000, 900, 77, 5000, 1000], 8, 2, 128, 16, device, seed=1)
    want = run(ext, case)
    for _ in range(3):
        held = [torch.full((n,), NAN, device=device) for n in (256, 65536, 1 << 20, 1 << 22, 12 << 20)]
        torch.cuda.synchronize()
        del held
        assert torch.equal(run(ext, case), want)


def test_empty_calls(ext, device):
    k = torch.zeros(4, 16, 2, 64, dtype=BF16, device=device)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    table = torch.zeros(0, 3, dtype=torch.int32, device=device)
    assert ext.paged_attention(torch.zeros(0, 1, 4, 64, dtype=BF16, device=device), k, k, table, ints()).shape == (0, 1, 4, 64)
    table = torch.zeros(2, 3, dtype=torch.int32, device=device)
    assert ext.paged_attention(torch.zeros(2, 0, 4, 64, dtype=BF16, device=device), k, k, table, ints(1, 1)).shape == (2, 0, 4, 64)
    q = torch.ones(3, 4, 64, dtype=BF16, device=device)
    out = torch.full_like(q, 3.0)
    ext.paged_attention(q, k, k, table, ints(1, 1), starts=ints(0, 0, 0), out=out)
    assert bool((out == 3.0).all())
    # no entries in the table: no token sees a key
    out = ext.paged_attention(torch.ones(2, 1, 4, 64, dtype=BF16, device=device), k, k, table[:, :0], ints(5, 5))
    assert bool((out == 0).all())


def test_refusals(ext, device):
    k = torch.zeros(4, 16, 2, 64, dtype=BF16, device=device)
    q = torch.zeros(2, 1, 4, 64, dtype=BF16, device=device)
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device=device), torch.ones(2, dtype=torch.int32, device=device)
    good = dict(query=q, cache_k=k, cache_v=k, page_table=table, seq_lens=lens)
    ext.paged_attention(**good)
    bad = [
        (dict(query=q.float()), "bfloat16"), (dict(query=q.cpu()), "CUDA tensor"), (dict(query=q[0]), r"\[B, T, Hq, D\]"),
        (dict(query=torch.zeros(3, 1, 4, 64, dtype=BF16, device=device)), "a row for every sequence"),
        (dict(query=torch.zeros(2, 1, 3, 64, dtype=BF16, device=device)), "head ratio"),
        (dict(query=torch.zeros(2, 1, 34, 64, dtype=BF16, device=device)), "head ratio"),
        (dict(query=torch.zeros(2, 1, 4, 32, dtype=BF16, device=device)), "head size"),
        (dict(query=torch.zeros(2, 4, 1, 65, dtype=BF16, device=device).transpose(1, 2)[..., 1:]), "16 bytes"),
        (dict(cache_v=k[:3]), "equal layout"), (dict(cache_k=k.transpose(1, 2), cache_v=k.transpose(1, 2)), "contiguous"),
        (dict(cache_k=torch.zeros(4, 24, 2, 64, dtype=BF16, device=device), cache_v=torch.zeros(4, 24, 2, 64, dtype=BF16, device=device)), "multiple of 16"),
        (dict(page_table=table.long()), "int32"), (dict(page_table=table.t()), "contiguous rows"), (dict(seq_lens=lens.long()), "int32"),
        (dict(seq_lens=lens[:1]), r"\[B\]"), (dict(starts=torch.zeros(2, dtype=torch.int32, device=device), query=q[:, 0]), r"\[B \+ 1\]"),
        (dict(out=torch.zeros(2, 1, 4, 32, dtype=BF16, device=device)), "shaped like query"),
        (dict(out=torch.zeros(2, 1, 4, 64, device=device)), "bfloat16"), (dict(out=q[:1].clone().expand(2, 1, 4, 64)), "places of their own"),
        (dict(cache_k=k[:1].expand(4, 16, 2, 64), cache_v=k[:1].expand(4, 16, 2, 64)), "places of their own"),
    ]
    for change, words in bad:
        with pytest.raises(RuntimeError, match=words):
            ext.paged_attention(**{**good, **change})
