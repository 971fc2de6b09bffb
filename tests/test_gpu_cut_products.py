"""Products that are cut among the pairs of CTAs, each asserted to be cut by the scratch it asks for, against
float64 on the same half-precision inputs.

Tolerances as in the other tests of the products: a float32 sum is off by at most 2^-18 of the sum of its
products' absolute values (one rounding per 16 products, of partial sums that random signs keep near the
square root of their number), the result by half a step."""

import ctypes as C

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

ACC = 2.0**-18
BF = torch.bfloat16


def _rand(seed, *shape, scale=1.0, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _scratch(rows, n, k, what, gated=False, dtype=BF):
    """Bytes that the product called ``what`` (fwd, dx, dw) asks for to be cut, without what lies before it."""
    from kvstreams import _native as N

    P = 0x10000
    a = N.KvsLinearArgs(x=P, weight=P, ld_x=k, ld_w=k, ld_out=n, rows=rows, n=n, k=k, dtype=N.DTYPE_CODE[dtype])
    if gated:
        a.weight_up, a.ld_w_up, a.pre, a.ld_pre = P, k, P, 2 * n
    if what == "fwd":
        return N.lib().kvs_linear_scratch_bytes(C.byref(a))
    size = lambda **kw: N.lib().kvs_linear_backward_scratch_bytes(  # noqa: E731
        C.byref(a), C.byref(N.KvsLinearGrads(gy=P, ld_gy=n, ld_dx=k, ld_dw=k, **kw)))
    return size(**({"dx": P} if what == "dx" else {"dw": P, "dw_up": P if gated else None})) - size()


def _near(got, want, bound, what):
    fi = torch.finfo(got.dtype)
    err = (got.double() - want).abs() - (want.abs() * fi.eps / 2 * 1.01 + bound + fi.tiny * fi.eps)
    assert err.max().item() <= 0, (what, err.max().item())


@pytest.mark.parametrize("rows,n,k", [(262153, 64, 64), (40001, 1, 4096), (33000, 16, 4096), (131079, 1001, 520)])
def test_weight_gradients_of_narrow_layers(rows, n, k):
    """Few tiles and very many rows: every pair of CTAs takes a share of the rows."""
    from kvstreams import ops

    assert _scratch(rows, n, k, "dw") > 0
    x, gy, w = _rand(1, rows, k), _rand(2, rows, n), _rand(3, n, k)
    dx, dw, db = ops.linear_backward(gy, x, w, bias_grad=True)
    gd, xd = gy.double(), x.double()
    _near(dw, gd.t() @ xd, gd.abs().t() @ xd.abs() * ACC, "dw")
    _near(db, gd.sum(0), gd.abs().sum(0) * ACC, "db")
    again = ops.linear_backward(gy, x, w, bias_grad=True)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))
