"""The distillation loss does not change when a row's logits are shifted together, and is as accurate far
from zero as near it.

Tolerances: a term is p (log p - (x - m) / T + log S), m the row's largest.  x - m is exact up to a rounding of its
own size; log S, log p and the quotients carry a few float32 roundings of their size, and the sums' 2^x and S
2^-21: four ulps, 2^-21, of 1 + |x - m| / T + log S + |log p|, weighted by p, which sums to 1."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab,top", [(300, 900, 20), (40, 5000, 64), (3, 50001, 64), (2, 128256, 300)])
@pytest.mark.parametrize("T", [1.0, 0.01])
@pytest.mark.parametrize("shift", [0.0, 1e4, -1e4, 1e6])
def test_shifted_logits(rows, vocab, top, T, shift):
    from kvstreams import ops

    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, vocab, generator=g, device="cuda") * (2.5 * T) + shift
    near = x.double() + torch.randn(rows, vocab, generator=g, device="cuda", dtype=torch.float64) * (0.1 * T)
    t, ids = near.topk(top, dim=-1)
    t = (t - t[:, :1]).float()
    loss, lse = ops.distill(x, ids, t, T)
    lp = torch.log_softmax(t.double() / T, -1)
    lq = torch.log_softmax(x.double() / T, -1).gather(1, ids)
    want = (lp.exp() * (lp - lq)).sum(-1)
    size = 1 + (x.double().amax(-1) - x.double().gather(1, ids).amin(-1)) / T + lq.abs().amax(-1) + lp.abs().amax(-1)
    assert ((loss.double() - want).abs() <= 2.0**-21 * size).all()
    assert (loss >= -2.0**-20).all()  # p sums to 1 over the slots and q over the vocabulary
    wlse = torch.logsumexp(x.double() / T, -1)
    assert ((lse.double() - wlse).abs() <= 2.0**-22 * (wlse.abs() + 16)).all()
