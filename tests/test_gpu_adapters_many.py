"""Low-rank adapters beside the product of many rows: the tests of test_gpu_adapters.py at sizes that this product takes (each test asks which one does),
and what a rounding of the low-rank factor would cost.

Tolerance: as there."""
import ctypes as C

import pytest
import torch

from test_gpu_adapters import BF16, check, make, spread

pytestmark = pytest.mark.gpu
FEW, MANY = 0, 1
# (rows, K, N): the first factor row by row (up to 512) and by tiles of rows beyond; the last tile of 256 rows and of 256 columns half empty
SIZES = [(500, 264, 2056), (2049, 264, 520)]
RANKS = [8, 16, 24, 32, 40, 64, 72, 104, 128]


def takes(capi, c):
    rows, K = c["x"].shape
    a = capi.AdapterLinearArgs(x=c["x"].data_ptr(), w=c["w"].data_ptr(), a=c["a"].data_ptr(), b=c["b"].data_ptr(), index=c["index"].data_ptr(), out=c["x"].data_ptr(), rows=rows, x_st=K,
                               out_st=c["w"].shape[0], K=K, N=c["w"].shape[0], rank=c["a"].shape[1], adapters=c["a"].shape[0])
    return capi.load().l3ci_adapter_linear_kernel_choice(C.byref(a))


def make_many(capi, device, rows, K, N, rank, adapters, index, seed=0):
    c = make(device, rows, K, N, rank, adapters, index, seed)
    assert takes(capi, c) == MANY
    return c


@pytest.mark.parametrize("rank", RANKS)
@pytest.mark.parametrize("rows,K,N", SIZES)
@pytest.mark.parametrize("run", [1, 90])
def test_ranks(ext, capi, device, rank, rows, K, N, run):
    c = make_many(capi, device, rows, K, N, rank, 5, spread(rows, 5, run), seed=rank + run)
    check(ext.adapter_linear(**c), c)


@pytest.mark.parametrize("rows,K,N", SIZES + [(1000, 520, 1000), (257, 64, 8192), (4000, 1032, 264)])
def test_as_many_adapters_as_a_tile_has_rows(ext, capi, device, rows, K, N):
    c = make_many(capi, device, rows, K, N, 24, 300, [r * 7 % 300 for r in range(rows)], seed=rows)
    check(ext.adapter_linear(**c), c)


@pytest.mark.parametrize("rank", [8, 40, 128])
@pytest.mark.parametrize("rows,K,N", SIZES)
def test_an_adapter_that_is_no_number_stays_with_its_rows(ext, capi, device, rank, rows, K, N):
    # neighbouring rows have three adapters and none; of two of them a or b is no number in places
    c = make_many(capi, device, rows, K, N, rank, 3, [r % 4 - 1 for r in range(rows)], seed=rows + rank)
    clean = ext.adapter_linear(**c)
    check(clean, c)
    c["a"][1, rank - 3, 5], c["b"][2, 7, rank - 1], c["b"][2, N - 2, 0] = float("nan"), float("inf"), float("nan")
    got = ext.adapter_linear(**c)
    assert torch.equal(got[0::4], clean[0::4]) and torch.equal(got[1::4], clean[1::4]), "rows without an adapter, and of the first one"
    assert torch.isnan(got[2::4]).all(), "a value of z that is no number meets every column"
    third = torch.ones(N, dtype=torch.bool, device=device)
    third[7] = third[N - 2] = False
    assert torch.equal(got[3::4][:, third], clean[3::4][:, third]) and not torch.isfinite(got[3::4][:, ~third]).any()


@pytest.mark.parametrize("rows,K,N", SIZES)
def test_rows_and_tiles_without_an_adapter(ext, capi, device, rows, K, N):
    none = (-1, 4, 2 ** 31 - 1, -2 ** 31)
    c = make_many(capi, device, rows, K, N, 16, 4, [none[r % 4] if r < 300 or r % 3 else r % 4 for r in range(rows)], seed=rows)
    want = ext.adapter_linear(**c)
    check(want, c)
    for _ in range(3):       # what their part of the scratch held before is nobody's
        held = [torch.full((n,), float("nan"), device=device) for n in (256, 4096, 65536, 1 << 18, 1 << 20)]
        torch.cuda.synchronize()
        del held
        assert torch.equal(ext.adapter_linear(**c), want)
    c["index"].fill_(-1)
    c["a"].fill_(float("nan")), c["b"].fill_(float("inf"))
    check(ext.adapter_linear(**{**c, "a": torch.zeros_like(c["a"]), "b": torch.zeros_like(c["b"])}), {**c, "a": torch.zeros_like(c["a"]), "b": torch.zeros_like(c["b"])})
    assert torch.isfinite(ext.adapter_linear(**c)).all()
    none = make_many(capi, device, rows, K, N, 16, 0, [0] * rows, seed=rows)
    check(ext.adapter_linear(**none), none)


@pytest.mark.parametrize("rows,K,N", SIZES)
def test_same_bits_on_another_stream_and_in_graphs_at_once(ext, capi, device, rows, K, N):
    c = make_many(capi, device, rows, K, N, 40, 6, spread(rows, 6, 50), seed=rows)
    want = ext.adapter_linear(**c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ext.adapter_linear(**c)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, other)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ext.adapter_linear(**c))
        graphs.append(g)
    c["index"].copy_(c["index"].flip(0))
    want = ext.adapter_linear(**c)
    check(want, c)
    torch.cuda.synchronize()
    for _ in range(10):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


@pytest.mark.parametrize("rank", [16, 40])
@pytest.mark.parametrize("rows,K,N,product", [(40, 264, 520, FEW), (500, 264, 2056, MANY), (2049, 264, 520, MANY)])
def test_the_low_rank_factor_keeps_more_than_eight_bits(ext, capi, device, rank, rows, K, N, product):
    # w = 0, and z = u + 2^-8 v of bf16 u and v in [1, 2): 16 bits.  Pairs of ranks share u and meet b = 1 and -1, so that the results are the sums of
    # 2^-8 (v - v'), of which a z of eight bits keeps nothing.  All terms are multiples of 2^-15, all sums below 2^7: 32 bits hold them, and the
    # results are off by their rounding; 2^-17 of the sum of |z b|, half of what two bf16 may lose of z, is allowed beside it.
    g = torch.Generator().manual_seed(rank + rows)
    c = make(device, rows, K, N, rank, 3, spread(rows, 3), seed=1)
    assert takes(capi, c) == product
    eighths = lambda *s: 1 + torch.randint(0, 128, s, generator=g) / 128  # noqa: E731
    c["scales"] = None
    c["w"].zero_(), c["x"].zero_(), c["a"].zero_()
    c["x"][:, 0], c["x"][:, K - 1] = 1.0, 2.0 ** -8
    c["a"][:, :, 0] = eighths(3, rank // 2).repeat_interleave(2, dim=1).to(BF16).to(device)
    c["a"][:, :, K - 1] = eighths(3, rank).to(BF16).to(device)
    sign = torch.tensor([1.0, -1.0], device=device).repeat(rank // 2).to(BF16)
    c["b"].copy_(sign.expand_as(c["b"]))
    got = ext.adapter_linear(**c).double()
    z = (c["a"][:, :, 0].double() + 2.0 ** -8 * c["a"][:, :, K - 1].double())
    want = torch.zeros(rows, dtype=torch.float64, device=device)
    mine = c["index"] >= 0
    want[mine] = (z * sign.double()).sum(1)[c["index"][mine].long()]
    bound = want.abs() * 2 ** -8 + 2 ** -17 * z.sum(1).max()
    assert bool(((got - want[:, None]).abs() <= bound[:, None]).all())
    eight = (z.to(BF16).double() * sign.double()).sum(1)[c["index"][mine].long()]
    assert bool(((eight - want[mine]).abs() > bound[mine]).any()), "a z of eight bits would be seen"
