"""What the entry points of paged caches and adapters refuse, at the C ABI and before any CUDA call (no GPU)."""
import ctypes as C

FAKE = 0x1000   # never dereferenced


def call(capi, name, struct, good, **change):
    return getattr(capi.load(), name)(C.byref(struct(**{**good, **change})))


def test_paged_rope(capi):
    good = dict(qkv=FAKE, freq_table=FAKE, q_out=FAKE, cache_k=FAKE, cache_v=FAKE, page_table=FAKE, positions=FAKE, qkv_sb=512, qkv_st=512, q_st=256, freq_rows=8,
                pages=4, cache_sp=2048, cache_st=128, table_st=2, B=2, T=1, Hq=4, Hkv=2, D=64, page_size=16, max_pages=2, eps=1e-5)
    go = lambda **kw: call(capi, "l3ci_rot_embed_paged_kv_cache", capi.PagedRopeArgs, good, **kw)  # noqa: E731
    for bad in (dict(qkv=None), dict(freq_table=None), dict(q_out=None), dict(cache_k=None), dict(cache_v=None), dict(page_table=None), dict(positions=None),
                dict(q_norm=FAKE), dict(k_norm=FAKE), dict(B=-1), dict(T=-1), dict(Hq=0), dict(Hkv=0), dict(D=0), dict(page_size=0), dict(max_pages=-1), dict(pages=-1),
                dict(freq_rows=-1), dict(starts=FAKE, rows=-1), dict(q_st=192), dict(starts=FAKE, rows=2 ** 31)):
        assert go(**bad) == capi.ERR_INVALID, bad
    for bad in (dict(D=60), dict(D=264)):
        assert go(**bad) == capi.ERR_UNSUPPORTED, bad
    for bad in (dict(qkv=FAKE + 2), dict(q_out=FAKE + 8), dict(cache_k=FAKE + 2), dict(cache_v=FAKE + 2), dict(freq_table=FAKE + 4), dict(q_norm=FAKE + 2, k_norm=FAKE),
                dict(qkv_st=516), dict(qkv_sb=4), dict(q_st=260), dict(cache_sp=2052), dict(cache_st=132)):
        assert go(**bad) == capi.ERR_ALIGNMENT, bad
    for nothing in (dict(B=0), dict(T=0), dict(starts=FAKE, rows=0)):
        assert go(**nothing) == capi.OK, nothing
    assert capi.load().l3ci_rot_embed_paged_kv_cache(None) == capi.ERR_INVALID


def test_paged_attention(capi):
    good = dict(q=FAKE, cache_k=FAKE, cache_v=FAKE, out=FAKE, page_table=FAKE, seq_lens=FAKE, q_sb=256, q_st=256, q_sh=64, o_sb=256, o_st=256, o_sh=64, pages=4,
                cache_sp=2048, cache_st=128, table_st=2, B=2, T=1, Hq=4, Hkv=2, D=64, page_size=16, max_pages=2)
    go = lambda **kw: call(capi, "l3ci_paged_attention", capi.PagedAttentionArgs, good, **kw)  # noqa: E731
    for bad in (dict(q=None), dict(cache_k=None), dict(cache_v=None), dict(out=None), dict(page_table=None), dict(seq_lens=None), dict(B=-1), dict(T=-1), dict(Hq=0),
                dict(Hkv=0), dict(page_size=0), dict(max_pages=-1), dict(pages=-1), dict(starts=FAKE, rows=-1), dict(max_pages=2 ** 30), dict(pages=2 ** 31),
                dict(starts=FAKE, rows=2 ** 31), dict(starts=FAKE, rows=2 ** 22, max_pages=2 ** 18)):
        assert go(**bad) == capi.ERR_INVALID, bad
    for bad in (dict(D=96), dict(Hq=5), dict(Hq=34), dict(page_size=24), dict(page_size=8)):
        assert go(**bad) == capi.ERR_UNSUPPORTED, bad
    for bad in (dict(q=FAKE + 2), dict(out=FAKE + 8), dict(cache_k=FAKE + 2), dict(cache_v=FAKE + 2), dict(q_st=260), dict(q_sh=60), dict(o_st=4), dict(cache_sp=2052),
                dict(cache_st=132)):
        assert go(**bad) == capi.ERR_ALIGNMENT, bad
    for nothing in (dict(B=0), dict(T=0), dict(starts=FAKE, rows=0)):
        assert go(**nothing) == capi.OK, nothing
    lib = capi.load()
    assert lib.l3ci_paged_attention(None) == capi.ERR_INVALID and lib.l3ci_paged_attention_scratch_bytes(None) == 0
    for bad in (dict(D=96), dict(q=None), dict(B=0)):
        assert lib.l3ci_paged_attention_scratch_bytes(C.byref(capi.PagedAttentionArgs(**{**good, **bad}))) == 0


def test_adapter_linear(capi):
    good = dict(x=FAKE, w=FAKE, a=FAKE, b=FAKE, index=FAKE, out=FAKE, rows=2, x_st=64, out_st=32, K=64, N=32, rank=16, adapters=3)
    go = lambda **kw: call(capi, "l3ci_adapter_linear", capi.AdapterLinearArgs, good, **kw)  # noqa: E731
    for bad in (dict(x=None), dict(w=None), dict(a=None), dict(b=None), dict(index=None), dict(out=None), dict(rows=-1), dict(rows=2 ** 31), dict(K=0), dict(N=-8),
                dict(rank=0), dict(adapters=-1), dict(x_st=0), dict(out_st=24)):
        assert go(**bad) == capi.ERR_INVALID, bad
    for bad in (dict(rank=12), dict(rank=136)):
        assert go(**bad) == capi.ERR_UNSUPPORTED, bad
    for bad in (dict(x=FAKE + 2), dict(w=FAKE + 2), dict(a=FAKE + 2), dict(b=FAKE + 8), dict(out=FAKE + 2), dict(K=60), dict(N=36), dict(x_st=68), dict(out_st=36)):
        assert go(**bad) == capi.ERR_ALIGNMENT, bad
    for nothing in (dict(rows=0), dict(N=0)):
        assert go(**nothing) == capi.OK, nothing
    lib = capi.load()
    need = lib.l3ci_adapter_linear_scratch_bytes(C.byref(capi.AdapterLinearArgs(**good)))
    assert need > 0
    for bad in (dict(), dict(scratch=FAKE, scratch_bytes=need - 1), dict(scratch=FAKE + 4, scratch_bytes=need)):
        assert go(**bad) == capi.ERR_SCRATCH, bad
    assert lib.l3ci_adapter_linear(None) == capi.ERR_INVALID and lib.l3ci_adapter_linear_scratch_bytes(None) == 0
