"""The layer products (kvs_linear / kvs_linear_backward, plain and gated) against float64 on the
same half-precision inputs.

Tolerances.  A forward output is a float32 sum of k exact products (a bf16 or fp16 product is exact
in float32) plus bias, activation and residual, rounded once.  The sum's error is at most
k * 2^-24 * sum|x w| and in practice far less: ACC = 2^-18 * sum|x||w| (64 ulps of the absolute sum)
bounds it up to k = 14344: one rounding per 16 products, 900 of them, each of a partial sum that the
random signs keep near sqrt(k) = 120 where the absolute sum is near 0.6 k.  The activations add a few
float32 ulps (covered by the same term) and the final rounding eps / 2 of the value.  A backward output
is a sum of products of two rounded operands: dz carries half a step of its own (eps / 2) and, with an
activation, the rounding of the kept pre-activation (2^-24, or half a step of the operands' type) times
the activation's curvature; the bound is that share of the absolute sum.  The absolute sums are
computed in float64 beside the result."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

ACT = {None: lambda z: z, "relu": torch.relu, "silu": F.silu, "gelu": F.gelu}
# largest |act'| and |act''| (silu 1.10 / 0.5, gelu 1.13 / 0.80 = 2 phi(0)); a pre-activation off by
# delta changes act' by at most curv * delta.  relu's derivative jumps at 0, which a rounding to
# nearest never crosses: a sum of the other sign would have to be below the smallest subnormal.
SLOPE = {None: (1.0, 0.0), "relu": (1.0, 0.0), "silu": (1.1, 0.5), "gelu": (1.13, 0.8)}
ACC = 2.0 ** -18

# enough K blocks and few enough tiles that the last ones are cut among the pairs of CTAs: fewer tiles
# than pairs, and a round of them over; ragged in every index
CUT = [(600, 1500, 14344), (520, 1001, 14344), (2560, 2305, 4104), (4000, 2560, 4104), (2560, 2304, 4104)]


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _rand(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _near(got, want, bound, dtype, what):
    """|got - want| <= half a step of want + bound (+ the smallest subnormal of the type)."""
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    err = (got.double() - want).abs() - (want.abs() * _half(dtype) * 1.01 + bound + tiny)
    assert err.max().item() <= 0, (what, err.max().item())


SIZES = [(1, 1, 8), (1, 4096, 512), (3, 129, 72), (64, 256, 64), (130, 255, 136), (257, 513, 200), (300, 1000, 1032),
         (777, 130, 4096)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("rows,n,k", SIZES)
def test_linear_forward(rows, n, k, act, dtype):
    from kvstreams import ops

    g = torch.Generator(device="cuda").manual_seed(rows * 7 + n + k)
    x, w, b, r = _rand(g, rows, k, dtype=dtype), _rand(g, n, k, scale=0.1, dtype=dtype), _rand(g, n, dtype=dtype), _rand(g, rows, n, dtype=dtype)
    z0 = x.double() @ w.double().t()
    mass = (x.double().abs() @ w.double().abs().t()) * ACC
    for bias, res, pdt in ((None, None, torch.float32), (b, r, torch.float32), (b, None, dtype)):
        pre = ops.pre_buffer(x, n, pdt)
        y = ops.linear(x, w, bias=bias, residual=res, activation=act, pre=pre)
        z = z0 if bias is None else z0 + bias.double()
        want = ACT[act](z) if res is None else ACT[act](z) + res.double()
        extra = mass * 2 + (z.abs() + 1) * 2.0 ** -20
        _near(pre, z, extra, pdt, "pre")
        _near(y, want, extra, dtype, "y")
        assert torch.equal(y, ops.linear(x, w, bias=bias, residual=res, activation=act))  # pre changes nothing


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("keep_half", [False, True])
@pytest.mark.parametrize("rows,n,k", SIZES)
def test_linear_backward(rows, n, k, keep_half, act, dtype):
    from kvstreams import ops

    g = torch.Generator(device="cuda").manual_seed(rows * 5 + n + k)
    x, w, b, gy = _rand(g, rows, k, dtype=dtype), _rand(g, n, k, scale=0.1, dtype=dtype), _rand(g, n, dtype=dtype), _rand(g, rows, n, dtype=dtype)
    pre = ops.pre_buffer(x, n, dtype if keep_half else torch.float32)
    ops.linear(x, w, bias=b, activation=act, pre=pre)
    dx, dw, db = ops.linear_backward(gy, x, w, pre=pre, activation=act, bias_grad=True)
    xd, wd, bd = (t.double().requires_grad_() for t in (x, w, b))
    z = F.linear(xd, wd, bd)
    want = torch.autograd.grad(ACT[act](z), [xd, wd, bd], gy.double())
    # the derivative is taken at the kept pre-activation, half a step of its type from z
    slope, curv = SLOPE[act]
    h, hp = _half(dtype), _half(pre.dtype)
    mass = (x.double().abs() @ w.double().abs().t() + b.double().abs()) * ACC + 2.0 ** -20
    off = gy.double().abs() * (curv * (z.detach().abs() * hp + mass) + slope * (h + 2.0 ** -20))
    if act == "relu":  # z of either sign within the float32 sum's error of 0 may take either derivative
        off = off + gy.double().abs() * (z.detach().abs() < mass)
    big = gy.double().abs() * slope
    _near(dx, want[0], off @ w.double().abs() + big @ w.double().abs() * ACC, dtype, "dx")
    _near(dw, want[1], off.t() @ x.double().abs() + big.t() @ x.double().abs() * ACC, dtype, "dw")
    _near(db, want[2], off.sum(0) + big.sum(0) * ACC, dtype, "db")
    again = ops.linear_backward(gy, x, w, pre=pre, activation=act, bias_grad=True)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", None])
@pytest.mark.parametrize("keep_half", [False, True])
@pytest.mark.parametrize("rows,n,k", SIZES)
def test_gated_linear(rows, n, k, keep_half, act, dtype):
    from kvstreams import ops

    g = torch.Generator(device="cuda").manual_seed(rows * 3 + n + k)
    x, gh = _rand(g, rows, k, dtype=dtype), _rand(g, rows, n, dtype=dtype)
    wg, wu = _rand(g, n, k, scale=0.05, dtype=dtype), _rand(g, n, k, scale=0.05, dtype=dtype)
    pre = ops.pre_buffer(x, 2 * n, dtype if keep_half else torch.float32)
    h = ops.gated_linear(x, wg, wu, activation=act, pre=pre)
    dx, dwg, dwu = ops.gated_linear_backward(gh, x, wg, wu, pre, activation=act)
    xd, gd, ud = (t.double().requires_grad_() for t in (x, wg, wu))
    zg, zu = F.linear(xd, gd), F.linear(xd, ud)
    y = ACT[act](zg) * zu
    want = torch.autograd.grad(y, [xd, gd, ud], gh.double())
    zg, zu, y = zg.detach(), zu.detach(), y.detach()
    ax, ag, au = x.double().abs(), wg.double().abs(), wu.double().abs()
    mg, mu = ax @ ag.t() * ACC + 2.0 ** -20, ax @ au.t() * ACC + 2.0 ** -20  # float32 errors of g, u
    slope, curv = SLOPE[act]
    _near(pre[:, :n], zg, mg, pre.dtype, "gate")
    _near(pre[:, n:], zu, mu, pre.dtype, "up")
    _near(h, y, slope * mg * (zu.abs() + mu) + (zg.abs() * slope + mg) * mu + y.abs() * 2.0 ** -20, dtype, "h")
    assert torch.equal(h, ops.gated_linear(x, wg, wu, activation=act))
    hs, hp = _half(dtype), _half(pre.dtype)
    eg, eu = zg.abs() * hp + mg, zu.abs() * hp + mu  # how far the kept g, u are off
    gm = gh.double().abs()
    # dg = gh u act'(g): off by gh (eu slope + |u| curv eg), rounded (hs); du = gh act(g) likewise
    jump = (zg.abs() < mg).double() if act == "relu" else 0.0
    og = gm * (eu * slope + (zu.abs() + eu) * (curv * eg + jump + slope * (hs + 2.0 ** -20)))
    ou = gm * (slope * eg + (zg.abs() + eg) * slope * (hs + 2.0 ** -20))
    bg, bu = gm * (zu.abs() * slope + 1), gm * (zg.abs() * slope + 1)
    _near(dx, want[0], og @ ag + ou @ au + (bg @ ag + bu @ au) * ACC, dtype, "dx")
    _near(dwg, want[1], (og.t() + bg.t() * ACC) @ ax, dtype, "dwg")
    _near(dwu, want[2], (ou.t() + bu.t() * ACC) @ ax, dtype, "dwu")


@pytest.mark.parametrize("rows,n,k", CUT)
def test_cut_tiles(rows, n, k):
    """Products whose last tiles are cut along k: forward with every epilogue part, gated with its
    pre-activations, and both gradients, against float64; the same bits again, and without scratch
    (whole tiles: another order of the same sums) within the same bounds."""
    import ctypes as C

    from kvstreams import _native as N, ops

    dtype = BF = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    x, w, u = _rand(g, rows, k), _rand(g, n, k, scale=0.05), _rand(g, n, k, scale=0.05)
    b, r, gy = _rand(g, n), _rand(g, rows, n), _rand(g, rows, n)
    args = N.KvsLinearArgs(x=x.data_ptr(), weight=w.data_ptr(), ld_x=k, ld_w=k, ld_out=n, rows=rows, n=n, k=k,
                           dtype=N.KVS_BF16)
    assert N.lib().kvs_linear_scratch_bytes(C.byref(args)) > 0  # this size is cut
    ax, aw, au, ag = (t.double().abs() for t in (x, w, u, gy))
    z = x.double() @ w.double().t() + b.double()
    mass = (ax @ aw.t() + b.double().abs()) * ACC + 2.0 ** -20
    pre = ops.pre_buffer(x, n)
    y = ops.linear(x, w, b, r, "silu", pre=pre)
    _near(pre, z, mass, torch.float32, "pre")
    _near(y, F.silu(z) + r.double(), mass * 1.2 + 2.0 ** -19, BF, "y")
    assert torch.equal(y, ops.linear(x, w, b, r, "silu"))
    plain = torch.empty_like(y)
    args.out, args.bias, args.residual, args.ld_res = plain.data_ptr(), b.data_ptr(), r.data_ptr(), n
    args.activation = N.ACTIVATION_CODES["silu"]
    assert N.lib().kvs_linear(C.byref(args), N.stream_ptr(x.device)) == 0
    _near(plain, F.silu(z) + r.double(), mass * 1.2 + 2.0 ** -19, BF, "whole tiles")
    gp = ops.pre_buffer(x, 2 * n)
    h = ops.gated_linear(x, w, u, pre=gp)
    zg, zu = x.double() @ w.double().t(), x.double() @ u.double().t()
    mg, mu = ax @ aw.t() * ACC + 2.0 ** -20, ax @ au.t() * ACC + 2.0 ** -20
    _near(gp[:, :n], zg, mg, torch.float32, "gate")
    _near(gp[:, n:], zu, mu, torch.float32, "up")
    _near(h, F.silu(zg) * zu, 1.1 * mg * (zu.abs() + mu) + (1.1 * zg.abs() + mg) * mu + 2.0 ** -19, BF, "h")
    assert torch.equal(h, ops.gated_linear(x, w, u))
    dx, dw, db = ops.linear_backward(gy, x, w, bias_grad=True)
    gd = gy.double()
    _near(dx, gd @ w.double(), ag @ aw * ACC, BF, "dx")
    _near(dw, gd.t() @ x.double(), ag.t() @ ax * ACC, BF, "dw")
    again = ops.linear_backward(gy, x, w, bias_grad=True)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))
    gx, g1, g2 = ops.gated_linear_backward(gy, x, w, u, gp)
    again = ops.gated_linear_backward(gy, x, w, u, gp)
    assert all(torch.equal(p, q) for p, q in zip((gx, g1, g2), again))
    s = torch.sigmoid(zg)
    dg, du = gd * zu * s * (1 + zg * (1 - s)), gd * F.silu(zg)
    e = 2.0 ** -8 * 1.01  # the rounding of dg and du, and the float32 errors behind it
    _near(gx, dg @ w.double() + du @ u.double(), e * (dg.abs() @ aw + du.abs() @ au) + 2.0 ** -10, BF, "gated dx")
    _near(g1, dg.t() @ x.double(), e * dg.abs().t() @ ax + 2.0 ** -10, BF, "dw gate")
    _near(g2, du.t() @ x.double(), e * du.abs().t() @ ax + 2.0 ** -10, BF, "dw up")


@pytest.mark.parametrize("rows", [8, 600])
def test_gelu_over_its_range(rows):
    """x W^T with W the identity is exact, so the output is gelu itself rounded once.  The normal
    distribution's F is off by 7.5e-8 (its formula) and by three roundings of 2^-24 (1.8e-7), times |z|;
    fp16 rounds by 2^-11 relative, below its normal numbers by 2^-25."""
    from kvstreams import ops

    z = torch.linspace(-10, 10, rows * 512, device="cuda").to(torch.float16).view(rows, 512)
    w = torch.eye(512, device="cuda", dtype=torch.float16)
    want = F.gelu(z.double())
    bound = want.abs() * 2.0**-11 + z.double().abs() * 2.6e-7 + 2.0**-25
    assert ((ops.linear(z, w, activation="gelu").double() - want).abs() <= bound).all()
