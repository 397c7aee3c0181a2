"""Low-rank adapters beside a shared projection against the formula in 64 bits.

Tolerance: one rounding to bf16 (2^-8 of the result) and sums in 32 bits, whose K (and rank) terms are off by 2^-23 each at most, of the sum of
their sizes; the low-rank part passes through z, kept to 2^-16."""
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def make(device, rows, K, N, rank, adapters, index, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return dict(x=r(rows, K).to(BF16).to(device), w=(r(N, K) * K ** -0.5).to(BF16).to(device), a=(r(adapters, rank, K) * K ** -0.5).to(BF16).to(device),
                b=(r(adapters, N, rank) * rank ** -0.5).to(BF16).to(device), index=torch.tensor(index, dtype=torch.int32, device=device),
                scales=(0.5 + torch.rand(adapters, generator=g)).to(device))


def check(got, c, rows=slice(None), columns=slice(None)):
    want, size, low = paged.adapter_linear(c["x"].reshape(-1, c["x"].shape[-1]), c["w"], c["a"], c["b"], c["index"].cpu().view(-1), c.get("scales"))
    K, rank = c["x"].shape[-1], c["a"].shape[1]
    off = (got.reshape(want.shape).double() - want).abs()
    bound = want.abs() * 2 ** -8 + size * K * 2 ** -23 + low * ((K + rank) * 2 ** -23 + 2 ** -16)
    off, bound = off[rows][:, columns], bound[rows][:, columns]
    assert bool((off <= bound).all()), f"{(off / bound).max().item():.3g} of the bound"


def spread(rows, adapters, run=1):
    return [(r // run * 7 + 3) % (adapters + 1) - 1 for r in range(rows)]


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 31, 32, 33, 63, 64, 65, 100])
@pytest.mark.parametrize("K,N,rank", [(256, 384, 16), (512, 136, 8), (1024, 1000, 64), (200, 264, 40)])
def test_few_rows_of_many_requests(ext, device, rows, K, N, rank):
    c = make(device, rows, K, N, rank, 11, spread(rows, 11), seed=rows + K)
    check(ext.adapter_linear(**c), c)


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 48, 72, 104, 128])
@pytest.mark.parametrize("rows", [5, 300])
def test_ranks(ext, device, rank, rows):
    c = make(device, rows, 512, 256, rank, 3, spread(rows, 3, run=50 if rows > 64 else 1), seed=rank)
    check(ext.adapter_linear(**c), c)


@pytest.mark.parametrize("rows,run", [(130, 130), (257, 40), (1000, 333), (2049, 700), (600, 1)])
@pytest.mark.parametrize("K,N", [(512, 768), (264, 520)])
def test_many_rows(ext, device, rows, run, K, N):
    c = make(device, rows, K, N, 16, 9, spread(rows, 9, run), seed=rows)
    check(ext.adapter_linear(**c), c)


def test_sizes_of_a_model(ext, device):
    for rows, K, N, rank, run in ((3, 2048, 8192, 16, 1), (48, 8192, 2048, 32, 1), (1500, 2048, 8192, 64, 400)):
        c = make(device, rows, K, N, rank, 20, spread(rows, 20, run), seed=rows)
        check(ext.adapter_linear(**c), c)


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_rows_without_an_adapter_and_no_adapters_at_all(ext, device, rows):
    c = make(device, rows, 256, 128, 16, 4, [(-1, 4, 2 ** 31 - 1, -2 ** 31)[r % 4] for r in range(rows)], seed=rows)
    check(ext.adapter_linear(**c), c)
    c["a"].fill_(float("nan"))   # (of adapters that no row has nothing is read)
    c["b"].fill_(float("inf"))
    got = ext.adapter_linear(**c)
    assert torch.isfinite(got).all()
    none = make(device, rows, 256, 128, 16, 0, [0] * rows, seed=rows)
    check(ext.adapter_linear(**none), none)


@pytest.mark.parametrize("rows", [6, 40, 300])
def test_an_adapter_that_is_no_number_stays_with_its_rows(ext, device, rows):
    c = make(device, rows, 256, 128, 16, 3, [r % 3 for r in range(rows)], seed=rows)
    clean = ext.adapter_linear(**c)
    c["a"][1, 3, 5], c["b"][2, 7, 1] = float("nan"), float("inf")
    got = ext.adapter_linear(**c)
    assert torch.equal(got[0::3], clean[0::3]) and torch.isnan(got[1::3]).all()
    third = torch.ones(128, dtype=torch.bool, device=device)
    third[7] = False
    # its own rows may be summed in another order then (multiply-adds for tensor cores): any order is within the bound, the bits may differ
    check(got, c, slice(2, None, 3), third)
    assert not torch.isfinite(got[2::3][:, 7]).any()


@pytest.mark.parametrize("rows,K,N", [(5, 256, 128), (100, 256, 128), (600, 2048, 136), (1500, 256, 512)])
def test_scratch_that_holds_no_numbers(ext, device, rows, K, N):
    # rows without an adapter in every product's form: what their part of the scratch held before is nobody's
    c = make(device, rows, K, N, 16, 3, [-1 if r % 3 == 0 else r % 2 for r in range(rows)], seed=rows)
    want = ext.adapter_linear(**c)
    check(want, c)
    for _ in range(3):
        held = [torch.full((n,), float("nan"), device=device) for n in (256, 4096, 65536, 1 << 20)]
        torch.cuda.synchronize()
        del held
        assert torch.equal(ext.adapter_linear(**c), want)


def test_shapes_strides_and_default_scales(ext, device):
    c = make(device, 24, 320, 144, 32, 5, spread(24, 5), seed=4)
    wide = torch.zeros(24, 400, dtype=BF16, device=device)
    wide[:, 40:360] = c["x"]
    base = ext.adapter_linear(**c)
    got = ext.adapter_linear(**{**c, "x": wide[:, 40:360].view(4, 6, 320)})
    assert got.shape == (4, 6, 144) and torch.equal(got.view(24, 144), base)
    c["scales"] = None
    check(ext.adapter_linear(**c), c)
    empty = ext.adapter_linear(**{**c, "x": c["x"][:0], "index": c["index"][:0]})
    assert empty.shape == (0, 144)


def test_same_bits_on_another_stream_and_in_graphs(ext, device):
    for rows in (12, 500):
        c = make(device, rows, 512, 256, 16, 6, spread(rows, 6, 1 if rows < 64 else 90), seed=rows)
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
        torch.cuda.synchronize()
        for _ in range(10):
            graphs[0].replay()
            with torch.cuda.stream(side):
                graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_refusals(ext, device):
    c = make(device, 4, 64, 32, 16, 2, [0, 1, 0, -1])
    bad = [
        (dict(x=c["x"].float()), "bfloat16"), (dict(x=c["x"].cpu()), "CUDA tensor"), (dict(w=c["w"][:, :32]), r"\[N, K\]"), (dict(a=c["a"][:, :, :32]), r"\[adapters, rank, K\]"),
        (dict(b=c["b"][:, :16]), r"\[adapters, N, rank\]"), (dict(index=c["index"].long()), "int32"), (dict(index=c["index"][:3]), "one entry per row"),
        (dict(scales=c["scales"][:1]), "one entry per adapter"), (dict(w=c["w"].t().contiguous().t()), "contiguous"),
        (dict(a=c["a"][:, :12].contiguous(), b=c["b"][:, :, :12].contiguous()), "multiple of 8"),
        (dict(a=torch.zeros(2, 136, 64, dtype=BF16, device=device), b=torch.zeros(2, 32, 136, dtype=BF16, device=device)), "multiple of 8 up to 128"),
        (dict(x=c["x"].t().contiguous().t()), "one stride"), (dict(x=c["x"][:1].expand(4, 64)), "one stride"),
        (dict(w=c["w"][:30], b=c["b"][:, :30].contiguous()), "16-byte"),
    ]
    for change, words in bad:
        with pytest.raises(RuntimeError, match=words):
            ext.adapter_linear(**{**c, **change})
