"""Attention of chunks over a paged cache whose bounded waits run out: the kernel gives up in order, says so, and the next call is as before.

Nothing is lost or held up: the output warps wait for a block's run of keys, some 20 ms here, under a limit of 1 ms.  All entries of the table name the one
page there is, so that a sequence of 200 million keys needs no memory."""
import ctypes as C

import pytest
import torch

from paged_cases import BF16, attention_case

pytestmark = pytest.mark.gpu
LIMIT_NS = 1_000_000
PAGE = 16384


def long_call(capi, device, D, heads, status):
    """Arguments of one chunk of 16 tokens behind 12000 tiles of 128 keys for every block of the device, and the tensors they point to."""
    keys = torch.cuda.get_device_properties(device).multi_processor_count * 12000 * 128 // heads // PAGE * PAGE
    g = torch.Generator(device=device).manual_seed(D)
    k, v = (torch.randn(1, PAGE, heads, D, generator=g, device=device).to(BF16) for _ in range(2))
    q = torch.randn(1, 16, 16 * heads, D, generator=g, device=device).to(BF16)
    table, lens, out = torch.zeros(1, keys // PAGE, dtype=torch.int32, device=device), torch.tensor([keys], dtype=torch.int32, device=device), torch.zeros_like(q)
    a = capi.PagedAttentionArgs(q=q.data_ptr(), cache_k=k.data_ptr(), cache_v=v.data_ptr(), out=out.data_ptr(), page_table=table.data_ptr(), seq_lens=lens.data_ptr(),
                                status=status.data_ptr(), q_sb=q.stride(0), q_st=q.stride(1), q_sh=D, o_sb=q.stride(0), o_st=q.stride(1), o_sh=D, pages=1, cache_sp=k.stride(0),
                                cache_st=k.stride(1), table_st=table.stride(0), B=1, T=16, Hq=16 * heads, Hkv=heads, D=D, page_size=PAGE, max_pages=keys // PAGE,
                                stream=torch.cuda.current_stream().cuda_stream)
    a.scratch_bytes = capi.load().l3ci_paged_attention_scratch_bytes(C.byref(a))
    scratch = torch.zeros(a.scratch_bytes, dtype=torch.uint8, device=device)
    a.scratch = scratch.data_ptr()
    return a, (k, v, q, table, lens, out, scratch)


# (one head: one segment a block; five: blocks that go from one head's unit to the next, where what waits for the first to end gives up too)
@pytest.mark.parametrize("D,heads", [(64, 1), (128, 1), (128, 5)])
def test_waits_that_run_out_end_the_call_and_are_reported(ext, capi, device, D, heads):
    case = attention_case([40, 1, 300], [900, 77, 1000], 8, 2, D, 16, device, seed=D)
    go = lambda: ext.paged_attention(case.q, case.k, case.v, case.table, case.seq_lens, starts=case.starts_arg)  # noqa: E731
    want = go()
    status = torch.zeros(1, dtype=torch.int32, device=device)
    a, held = long_call(capi, device, D, heads, status)
    torch.cuda.synchronize()
    t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    with capi.device_wait_limit(LIMIT_NS):
        t0.record()
        assert capi.load().l3ci_paged_attention(C.byref(a)) == capi.OK
        t1.record()
        torch.cuda.synchronize()
    assert t0.elapsed_time(t1) < 1000.0
    assert int(status) == capi.ERR_DEVICE_WAIT
    assert torch.equal(go(), want)
    del held


def test_the_extension_reports_them_once(ext, capi, device):
    D, keys = 64, torch.cuda.get_device_properties(device).multi_processor_count * 12000 * 128 // PAGE * PAGE
    k, v = (torch.randn(1, PAGE, 1, D, device=device).to(BF16) for _ in range(2))
    q = torch.randn(1, 16, 16, D, device=device).to(BF16)
    table = torch.zeros(1, keys // PAGE, dtype=torch.int32, device=device)
    lens = torch.tensor([PAGE], dtype=torch.int32, device=device)
    want = ext.paged_attention(q, k, v, table, lens)
    assert ext.paged_attention_status(q) == capi.OK
    with capi.device_wait_limit(LIMIT_NS):
        ext.paged_attention(q, k, v, table, lens * (keys // PAGE))
        torch.cuda.synchronize()
    assert ext.paged_attention_status(q) == capi.ERR_DEVICE_WAIT
    assert ext.paged_attention_status(q) == capi.OK
    assert torch.equal(ext.paged_attention(q, k, v, table, lens), want) and ext.paged_attention_status(q) == capi.OK
