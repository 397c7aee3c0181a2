"""The attention half of a layer of a server, as it is used: projection with adapters, append to the paged cache, attention, projection with
adapters; sequences come in chunks and go on token by token.  Every call against its formula in 64 bits from the inputs that it was given, with
the tolerances of that call's own tests; and the whole in graphs, with and without programmatic launches, to the bit."""
from types import SimpleNamespace

import pytest
import torch

from oracle import inputs, paged
from oracle.rope import freqs_cis_reference
from paged_cases import BF16, NAN, table_of
from test_gpu_adapters import check as check_linear
from test_gpu_paged_attention import check as check_attention

pytestmark = pytest.mark.gpu


def make(device, totals, width, Hq, Hkv, D, page, adapters, rank, seed, norms=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(BF16).to(device)  # noqa: E731
    heads = (Hq + 2 * Hkv) * D
    table, pages = table_of(g, totals, page)
    low = lambda N, K: dict(w=r(N, K, scale=K ** -0.5), a=r(adapters, rank, K, scale=K ** -0.5), b=r(adapters, N, rank, scale=rank ** -0.5),  # noqa: E731
                            scales=(0.5 + torch.rand(adapters, generator=g)).to(device))
    m = SimpleNamespace(Hq=Hq, Hkv=Hkv, D=D, g=g, width=width, table=table.to(device), qkv=low(heads, width), proj=low(width, Hq * D),
                        freq=freqs_cis_reference(D, max(totals), **inputs.ROPE_CONFIG4).contiguous().to(device), norms={},
                        k=torch.full((pages, page, Hkv, D), NAN, dtype=BF16, device=device), v=torch.full((pages, page, Hkv, D), NAN, dtype=BF16, device=device))
    if norms:
        m.norms = dict(q_norm=(1 + 0.2 * torch.randn(D, generator=g)).to(BF16).to(device), k_norm=(1 + 0.2 * torch.randn(D, generator=g)).to(BF16).to(device))
    return m


def step(ext, m, x, index, positions, seq_lens, starts):
    qkv = ext.adapter_linear(x, m.qkv["w"], m.qkv["a"], m.qkv["b"], index, scales=m.qkv["scales"])
    q = ext.rot_embed_paged_kv_cache(qkv, m.freq, m.k, m.v, m.table, positions, m.Hq, m.Hkv, starts=starts, **m.norms)
    o = ext.paged_attention(q, m.k, m.v, m.table, seq_lens, starts=starts)
    y = ext.adapter_linear(o.flatten(-2), m.proj["w"], m.proj["a"], m.proj["b"], index, scales=m.proj["scales"])
    return qkv, q, o, y


def ints(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


def starts_of(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


@pytest.mark.parametrize("Hq,Hkv,D,norms", [(8, 2, 64, True), (4, 4, 128, False), (12, 2, 128, True)])
def test_sequences_in_chunks_and_then_token_by_token(ext, device, Hq, Hkv, D, norms):
    m = make(device, [170, 330, 40, 1], 256, Hq, Hkv, D, 16, adapters=3, rank=16, seed=D + Hq, norms=norms)
    positions, adapter = [0, 0, 0, 0], [1, -1, 2, 0]
    for new in ([100, 300, 1, 0], [60, 1, 1, 1], [1, 20, 30, 0], [1, 1, 1, 0], [0, 1, 1, 0]):
        starts, rows = starts_of(new), sum(new)
        x = torch.randn(rows, m.width, generator=m.g).to(BF16).to(device)
        index = ints([a for a, n in zip(adapter, new) for _ in range(n)], device)
        lens = [p + n for p, n in zip(positions, new)]
        qkv, q, o, y = step(ext, m, x, index, ints(positions, device), ints(lens, device), ints(starts, device))
        check_linear(qkv, dict(x=x, index=index, **m.qkv))
        want = paged.append(qkv, m.freq, m.k, m.v, m.table.cpu(), positions, starts, Hq, Hkv, **m.norms)
        for got, name in ((q, "q"), (m.k.flatten(0, 1), "k"), (m.v.flatten(0, 1), "v")):
            at, value, size = want[name]
            assert len(at) == rows and bool(((got[at].double() - value).abs() <= value.abs() * 2 ** -8 + size * 2 ** -20 + 1e-38).all()), name
        check_attention(o, SimpleNamespace(rows=q, k=m.k, v=m.v, table=m.table, seq_lens=ints(lens, device), starts=starts))
        check_linear(y, dict(x=o.flatten(-2), index=index, **m.proj))
        positions = lens
    assert positions == [162, 323, 34, 1]


@pytest.mark.parametrize("Hkv,D", [(2, 64), (4, 128)])
def test_the_dense_calls_on_the_same_rows(ext, capi, device, Hkv, D):
    # without norms the append's bits are those of the dense cache; both attentions are within the bound of the formula
    B, T, Hq = 2, 150, 8
    m = make(device, [T] * B, 128, Hq, Hkv, D, 16, adapters=1, rank=8, seed=D, norms=False)
    qkv = torch.randn(B, T, (Hq + 2 * Hkv) * D, generator=m.g).to(BF16).to(device)
    dense = [torch.zeros(B, T, Hkv, D, dtype=BF16, device=device) for _ in range(2)]
    want_q = ext.rot_embed_kv_cache(qkv, m.freq, *dense, 0, Hq, Hkv)
    q = ext.rot_embed_paged_kv_cache(qkv, m.freq, m.k, m.v, m.table, ints([0] * B, device), Hq, Hkv)
    assert torch.equal(q, want_q)
    for b in range(B):
        assert all(torch.equal(paged.rows_of(c, m.table[b], T), d[b]) for c, d in zip((m.k, m.v), dense))
    case = SimpleNamespace(rows=q.flatten(0, 1), k=m.k, v=m.v, table=m.table, seq_lens=ints([T] * B, device), starts=paged.uniform_starts(B, T))
    check_attention(ext.paged_attention(q, m.k, m.v, m.table, case.seq_lens), case)
    check_attention(capi.prefill_attention(q.transpose(1, 2), *(d.transpose(1, 2) for d in dense)).transpose(1, 2), case)


@pytest.mark.parametrize("programmatic", [True, False])
@pytest.mark.parametrize("new", [[1] * 5, [1, 90, 3, 1, 0]])
def test_two_captured_steps_at_once_give_the_bits_of_eager_ones(ext, capi, device, new, programmatic):
    repeats, rows, starts = 4, sum(new), starts_of(new)
    begin = [200, 31, 0, 7, 90]
    models, want = [], []
    for seed in (1, 2):
        m = make(device, [b + repeats * n + 1 for b, n in zip(begin, new)], 512, 8, 2, 128, 16, adapters=4, rank=32, seed=seed)
        m.k.normal_(), m.v.normal_()
        m.x = torch.randn(rows, m.width, generator=m.g).to(BF16).to(device)
        m.index = ints([(r // 3 + seed) % 5 - 1 for r in range(rows)], device)
        m.starts, m.new, m.begin = ints(starts, device), ints(new, device), ints(begin, device)
        m.positions, m.lens = m.begin.clone(), m.begin + m.new
        models.append(m)
        before = m.k.clone(), m.v.clone()
        positions, results = m.begin.clone(), []
        for _ in range(repeats):
            results.append(step(ext, m, m.x, m.index, positions, positions + m.new, m.starts)[-1].clone())
            positions = positions + m.new
        want.append((torch.stack(results), m.k.clone(), m.v.clone()))
        m.k.copy_(before[0]), m.v.copy_(before[1])
    graphs, side = [], torch.cuda.Stream()
    with capi.programmatic_launch(programmatic):
        for m in models:
            m.got, m.turn = torch.zeros(repeats, rows, m.width, dtype=BF16, device=device), torch.zeros(1, dtype=torch.int64, device=device)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = step(ext, m, m.x, m.index, m.positions, m.lens, m.starts)[-1]
                m.got.index_copy_(0, m.turn, y[None])
                m.positions.add_(m.new), m.lens.add_(m.new), m.turn.add_(1)
            graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(repeats):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    for m, (results, k, v) in zip(models, want):
        assert torch.equal(m.got, results)
        assert torch.equal(m.k.view(torch.int16), k.view(torch.int16)) and torch.equal(m.v.view(torch.int16), v.view(torch.int16))
