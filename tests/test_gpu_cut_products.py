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


def _off(t, shift):
    """A copy of ``t`` whose rows start ``shift`` elements into a wider buffer (1: misaligned too)."""
    wide = torch.full((t.shape[0], t.shape[1] + 13), 3.0, dtype=t.dtype, device=t.device)
    wide[:, shift:shift + t.shape[1]] = t
    return wide[:, shift:shift + t.shape[1]]


def _silu_grad(z):
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


# gated forwards: a whole round in front (160 units on 74 pairs), none (100), ragged columns
@pytest.mark.parametrize("rows,n,k", [(4000, 1153, 4104), (2560, 1160, 8200), (900, 3001, 4104)])
def test_gated_forward(rows, n, k):
    from kvstreams import ops

    assert _scratch(rows, n, k, "fwd", gated=True) > 0
    x, w, u = _rand(1, rows, k), _rand(2, n, k, scale=0.02), _rand(3, n, k, scale=0.02)
    pre = ops.pre_buffer(x, 2 * n)
    h = ops.gated_linear(x, w, u, pre=pre)
    xd, wd, ud = x.double(), w.double(), u.double()
    zg, zu = xd @ wd.t(), xd @ ud.t()
    mg, mu = (xd.abs() @ wd.abs().t()) * ACC + 2.0**-20, (xd.abs() @ ud.abs().t()) * ACC + 2.0**-20
    _near(pre[:, :n], zg, mg, "gate")
    _near(pre[:, n:], zu, mu, "up")
    _near(h, F.silu(zg) * zu, 1.1 * mg * (zu.abs() + mu) + (1.1 * zg.abs() + mg) * mu + 2.0**-19, "h")
    for shift in (1, 8):
        assert torch.equal(ops.gated_linear(_off(x, shift), _off(w, shift), _off(u, shift)), h)
    out = _off(torch.zeros_like(h), 1)
    assert torch.equal(ops.gated_linear(x, w, u, out=out), h)


@pytest.mark.parametrize("rows,n,k", [(4000, 1153, 4104), (600, 1501, 14344)])
def test_forward_with_every_epilogue_part(rows, n, k):
    from kvstreams import ops

    assert _scratch(rows, n, k, "fwd") > 0
    x, w, b, r = _rand(1, rows, k), _rand(2, n, k, scale=0.02), _rand(3, n), _rand(4, rows, n)
    y = ops.linear(x, w, b, r, "gelu")
    z = x.double() @ w.double().t() + b.double()
    mass = (x.double().abs() @ w.double().abs().t() + b.double().abs()) * ACC
    _near(y, F.gelu(z) + r.double(), 1.2 * mass + 2.0**-19 * (1 + z.abs()), "y")
    for shift in (1, 8):
        assert torch.equal(ops.linear(_off(x, shift), _off(w, shift), b, _off(r, shift), "gelu"), y)
    res = _off(r, 1)
    assert torch.equal(ops.linear(x, w, b, res, "gelu", out=res), y)


@pytest.mark.parametrize("rows,n,k", [(4000, 5001, 2568), (520, 14337, 1000)])
def test_input_gradient(rows, n, k):
    from kvstreams import ops

    assert _scratch(rows, n, k, "dx") > 0
    x, w, gy = _rand(1, rows, k), _rand(2, n, k, scale=0.02), _rand(3, rows, n)
    dx, _, _ = ops.linear_backward(gy, x, w, need_dw=False)
    _near(dx, gy.double() @ w.double(), gy.double().abs() @ w.double().abs() * ACC, "dx")
    for shift in (1, 8):
        assert torch.equal(ops.linear_backward(_off(gy, shift), x, _off(w, shift), need_dw=False)[0], dx)


@pytest.mark.parametrize("rows,n,k", [(700, 5001, 2048), (1000, 9001, 520)])
def test_gated_input_gradient(rows, n, k):
    from kvstreams import ops

    assert _scratch(rows, n, k, "dx", gated=True) > 0
    x, w, u, gh = _rand(1, rows, k), _rand(2, n, k, scale=0.02), _rand(3, n, k, scale=0.02), _rand(4, rows, n)
    pre = _rand(5, rows, 2 * n, dtype=torch.float32)
    dx, _, _ = ops.gated_linear_backward(gh, x, w, u, pre, need_dw=False)
    g, v, gd = pre[:, :n].double(), pre[:, n:].double(), gh.double()
    dg, du = gd * v * _silu_grad(g), gd * F.silu(g)
    # dg and du are rounded to bf16 (half a step, 2^-8), behind float32 arithmetic
    eg, eu = dg.abs() * 2.0**-8 * 1.01 + (gd * v).abs() * 2.0**-20, du.abs() * 2.0**-8 * 1.01
    _near(dx, dg @ w.double() + du @ u.double(), eg @ w.double().abs() + eu @ u.double().abs(), "gated dx")
    got = ops.gated_linear_backward(_off(gh, 1), x, _off(w, 1), _off(u, 8), _off(pre, 1), need_dw=False)[0]
    assert torch.equal(got, dx)


@pytest.mark.parametrize("rows,n,k", [(8192, 1001, 520), (4000, 1153, 4104)])
def test_weight_gradient_of_odd_width(rows, n, k):
    """dz in rows of its own, an odd number of them reduced over."""
    from kvstreams import ops

    assert _scratch(rows, n, k, "dw") > 0
    x, w, gy = _rand(1, rows, k), _rand(2, n, k, scale=0.02), _rand(3, rows, n)
    _, dw, db = ops.linear_backward(gy, x, w, bias_grad=True, need_dx=False)
    gd, xd = gy.double(), x.double()
    _near(dw, gd.t() @ xd, gd.abs().t() @ xd.abs() * ACC, "dw")
    _near(db, gd.sum(0), gd.abs().sum(0) * ACC, "db")
    for shift in (1, 8):
        assert torch.equal(ops.linear_backward(_off(gy, shift), _off(x, shift), w, need_dx=False)[1], dw)


# two results in one list of units; with a whole round in front (180 units) and without (24)
@pytest.mark.parametrize("rows,n,k", [(8192, 1001, 520), (8200, 2305, 2056)])
def test_gated_weight_gradients(rows, n, k):
    from kvstreams import ops

    assert _scratch(rows, n, k, "dw", gated=True) > 0
    x, w, u, gh = _rand(1, rows, k), _rand(2, n, k, scale=0.02), _rand(3, n, k, scale=0.02), _rand(4, rows, n)
    pre = _rand(5, rows, 2 * n, dtype=torch.float32)
    _, dwg, dwu = ops.gated_linear_backward(gh, x, w, u, pre, need_dx=False)
    g, v, gd, xa = pre[:, :n].double(), pre[:, n:].double(), gh.double(), x.double().abs()
    dg, du = gd * v * _silu_grad(g), gd * F.silu(g)
    eg, eu = dg.abs() * 2.0**-8 * 1.01 + (gd * v).abs() * 2.0**-20, du.abs() * 2.0**-8 * 1.01
    _near(dwg, dg.t() @ x.double(), eg.t() @ xa, "dw gate")
    _near(dwu, du.t() @ x.double(), eu.t() @ xa, "dw up")
    # the same product in a graph, twice with other values, beside an eager call
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.gated_linear_backward(gh, x, w, u, pre, need_dx=False)
    for seed in (6, 7):
        gh.copy_(_rand(seed, rows, n))
        graph.replay()
        want = ops.gated_linear_backward(gh, x, w, u, pre, need_dx=False)
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
