"""The activations of the products, on their own: with W the identity the sum is exact, so the output is the
activation of a half-precision number, rounded once.

Tolerances: half a step of the value (eps / 2, and half the smallest subnormal below the normal numbers) and
what the float32 arithmetic in front of it is off, relative to the value:
gelu   z F(z), F(-|z|) = e t P(t): the formula 1.5e-7; e = 2^(c z^2) carries three roundings of 2^-24 of an exponent
       of z^2 / 2 natural units, and 2^-22 of its own; t a quotient good to 2 ulps and a rounding, 2^-22, which F
       takes up to three times (d log F / d log t < 3); Horner's steps, the products: ten roundings.  Together
       below 3 (z^2 / 2) 2^-24 + 2^-19.  For z > 0, F = 1 - F(-z) is nearer.
silu   z / (1 + 2^(-|z| log2 e)) or its mirror: the exponent carries two roundings of 2^-24 of |z| natural units, 2^x
       2^-22, the quotient 2 ulps, four roundings more: below 2 |z| 2^-24 + 2^-20, and below 2^-126 of the sigmoid
       the spacing 2^-149 of its subnormal numbers, |z| times."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def _all_between(lo, hi, dtype):
    """Every number of the type between lo and hi."""
    bits = torch.arange(1 << 16, dtype=torch.int32, device="cuda").to(torch.int16)
    v = bits.view(dtype)
    return v[torch.isfinite(v) & (v >= lo) & (v <= hi)]


def _applied(z, act, rows):
    """act of the numbers z through a product with the identity, ``rows`` rows at a time (8: weights streamed,
    600: pairs of CTAs)."""
    from kvstreams import ops

    eye = torch.eye(64, device="cuda", dtype=z.dtype)
    pad = -z.numel() % (rows * 64)
    zz = torch.cat([z, z.new_zeros(pad)]).view(-1, rows, 64)
    return torch.cat([ops.linear(part, eye, activation=act).flatten() for part in zz])[:z.numel()]


@pytest.mark.parametrize("rows", [8, 600])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gelu_to_a_rounding(dtype, rows):
    z = _all_between(-12.9, 12.9, dtype)
    got, zd = _applied(z, "gelu", rows).double(), z.double()
    # z F(z) in 64 bits without cancellation: F(z) = erfc(-z / sqrt 2) / 2
    want = zd * torch.special.erfc(-zd * 0.5**0.5) / 2
    fi = torch.finfo(dtype)
    rel = fi.eps / 2 + 1.5 * zd * zd * 2.0**-24 + 2.0**-19
    assert ((got - want).abs() <= want.abs() * rel + fi.tiny * fi.eps / 2).all()


@pytest.mark.parametrize("rows", [8, 600])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_silu_to_a_rounding(dtype, rows):
    """Down to where silu passes bf16's subnormal numbers, in the plain and the gated form."""
    from kvstreams import ops

    z = _all_between(-110, 110, dtype)
    got, zd = _applied(z, "silu", rows).double(), z.double()
    want = zd * torch.sigmoid(zd)
    fi = torch.finfo(dtype)
    rel = fi.eps / 2 + zd.abs() * 2.0**-23 + 2.0**-20
    bound = want.abs() * rel + fi.tiny * fi.eps / 2 + zd.abs() * 2.0**-149
    assert ((got - want).abs() <= bound).all()
    # the same with a factor of 1 (w_up picks a column of ones)
    eye = torch.eye(64, device="cuda", dtype=dtype)
    up = torch.zeros_like(eye)
    up[:, 63] = 1
    zz = torch.cat([z, z.new_zeros(-z.numel() % (rows * 63))]).view(-1, 63)
    x = torch.cat([zz, torch.ones_like(zz[:, :1])], 1)
    h = torch.cat([ops.gated_linear(part, eye, up) for part in x.split(rows)])[:, :63].reshape(-1)[:z.numel()]
    assert torch.equal(h.double(), got)


def test_silu_gradient_below_the_border():
    """gy silu'(z) = gy s (1 + z (1 - s)) where s is below 2^-126: dx of a product with the identity."""
    from kvstreams import ops

    z = torch.tensor([-80.0, -86.5, -87.5, -88.0, -88.5, -90.0, 0.0, 88.5], device="cuda").bfloat16()
    x = z.repeat(8, 8)
    w = torch.eye(64, device="cuda").bfloat16()
    pre = ops.pre_buffer(x, 64)
    ops.linear(x, w, activation="silu", pre=pre)
    gy = torch.full_like(x, 2.0)
    dx, _, _ = ops.linear_backward(gy, x, w, pre=pre, activation="silu")
    zd = x.double().requires_grad_()
    (want,) = torch.autograd.grad(F.silu(zd), [zd], gy.double())
    # dz is rounded to bf16, the product with the identity is exact; s good as in silu, 1 + z (1 - s) to 2^-22 of |z|
    fi = torch.finfo(torch.bfloat16)
    bound = want.abs() * (fi.eps / 2 + 2.0**-15) + fi.tiny * fi.eps + 200 * 2.0**-149
    assert ((dx.double() - want).abs() <= bound).all()
