"""How the products are dealt out (host side): a narrow layer's weight gradient over many rows stays cut
among the pairs of CTAs whatever the number of rows, up to the largest that the calls take."""

import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from kvstreams import _native as N

    return N.load_library()


def _dw_scratch(lib, rows, n, k):
    from kvstreams import _native as N

    P = 0x10000  # an aligned address that nothing reads
    ld = (n + 7) // 8 * 8
    a = N.KvsLinearArgs(x=P, weight=P, ld_x=k, ld_w=k, rows=rows, n=n, k=k, dtype=N.KVS_BF16)
    g = N.KvsLinearGrads(gy=P, dw=P, ld_gy=ld, ld_dw=k)
    return lib.kvs_linear_backward_scratch_bytes(C.byref(a), C.byref(g))


@pytest.mark.parametrize("n,k", [(64, 64), (1, 4096), (16, 4096), (1001, 520), (1, 8), (1024, 2048)])
def test_weight_gradients_of_narrow_layers_stay_cut(lib, n, k):
    sizes = [_dw_scratch(lib, rows, n, k) for rows in (1 << s for s in range(16, 31))]
    assert all(s > 0 for s in sizes)
    # more rows never leave fewer pairs at work
    assert sizes == sorted(sizes)
