"""Which product the adapters take, and that it can be asked for (no GPU: the rule for 148 SMs)."""
import ctypes as C

FEW, MANY = 0, 1


def test_which_product_a_call_takes(capi):
    fake = dict(x=4096, w=4096, a=4096, b=4096, index=4096, out=4096)
    lib = capi.load()
    choice = lambda rows, K, N, rank, **kw: lib.l3ci_adapter_linear_kernel_choice(C.byref(capi.AdapterLinearArgs(**{**fake, **dict(rows=rows, x_st=K, out_st=N, K=K, N=N, rank=rank, adapters=2), **kw})))  # noqa: E731
    assert [choice(r, 2048, 8192, 16) for r in (1, 8, 64, 6001)] == [FEW, FEW, FEW, MANY]
    assert choice(4, 2048, 8192, 12) == choice(4, 2048, 8192, 136) == choice(4, 2044, 8192, 16) == choice(-1, 64, 64, 8) == -1
    assert lib.l3ci_adapter_linear_kernel_choice(None) == -1
