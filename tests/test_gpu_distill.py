"""Distillation from a teacher's top logits (kvs_distill / kvs_distill_backward) against float64.

Tolerances: the loss is a float32 sum with weights p_j that sum to 1 of terms log p - x/T + lse, each
good to a few float32 ulps of |x/T| + |lse| + |log p| (2^-20 relative to 1 + that size is eight of them);
an entry of the gradient is g/T (q - p) with q = 2^(x s - lse s): the exponent's rounding makes q off by
2^-23 * (|x/T| + |lse|) relative, a few ulps more for the exponential; then one rounding to the output type."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _case(rows, vocab, top, dtype, seed, scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g, device="cuda", dtype=torch.float64) * scale).to(dtype)
    near = x.double() + torch.randn(rows, vocab, generator=g, device="cuda", dtype=torch.float64)
    t, ids = near.topk(top, dim=-1)
    t = t if dtype == torch.float64 else t.float()
    grad = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64).to(t.dtype)
    return x, ids, t.clone(), grad


def _exact(x, ids, t, grad, T):
    xd = x.double().requires_grad_()
    kept = (ids >= 0) & (t > -math.inf)
    logq = torch.log_softmax(xd / T, -1).gather(1, ids.clamp(min=0))
    lp = torch.log_softmax(torch.where(kept, t.double() / T, -1e300), -1)
    p = torch.where(kept, lp.exp(), 0.0)
    on = kept & (p > 0)
    loss = torch.where(on, p * (torch.where(on, lp, 0.0) - torch.where(on, logq, 0.0)), 0.0).sum(-1)
    (d,) = torch.autograd.grad(loss, [xd], grad.double())
    return loss.detach(), torch.logsumexp(x.double() / T, -1), d, p


def _check(x, ids, t, grad, T, out_dtype):
    from kvstreams import ops

    loss, lse = ops.distill(x, ids, t, T)
    d = ops.distill_backward(x, ids, t, lse, grad, T, out_dtype=out_dtype)
    want, wlse, wd, p = _exact(x, ids, t, grad, T)
    u = 2.0 ** -20 if x.dtype != torch.float64 else 2.0 ** -46
    size = 1 + wlse.abs() + (x.double() / T).nan_to_num(0, 0, 0).abs().amax(-1) + (t.double() / T).nan_to_num(0, 0, 0).abs().amax(-1)
    assert loss.dtype == lse.dtype == (torch.float64 if x.dtype == torch.float64 else torch.float32)
    assert ((loss.double() - want).abs() <= u * size).all()
    assert ((lse.double() - wlse).abs() <= u * size).all()
    q = torch.exp(x.double() / T - wlse[:, None])
    eps = torch.finfo(out_dtype).eps
    scale = (grad.double() / T)[:, None]
    has = torch.zeros_like(q).scatter_add_(1, ids.clamp(min=0), p)
    bound = scale * u * (q * size[:, None] + has) + wd.abs() * eps * 0.51 + torch.finfo(out_dtype).tiny * eps
    if out_dtype == torch.float16:
        bound = bound + 2.0 ** -25
    assert ((d.double() - wd).abs() <= bound).all(), ((d.double() - wd).abs() - bound).max().item()
    loss2, lse2 = ops.distill(x, ids, t, T)
    assert torch.equal(loss, loss2) and torch.equal(lse, lse2)
    return loss, lse, d


@pytest.mark.parametrize("dtype,out", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                       (torch.float32, torch.float16), (torch.bfloat16, torch.bfloat16),
                                       (torch.float16, torch.float16), (torch.float64, torch.float64)])
@pytest.mark.parametrize("rows,vocab,top,T", [(1, 1, 1, 1.0), (5, 104, 104, 0.7), (33, 1000, 20, 2.0),
                                              (9, 32003, 64, 1.0), (2, 128256, 128, 1.0), (3, 2049, 1024, 1.3),
                                              (700, 195, 7, 1.0), (1, 50001, 3, 1.0)])
def test_matches_float64(rows, vocab, top, T, dtype, out):
    _check(*_case(rows, vocab, top, dtype, rows + vocab), T, out)


def test_empty_slots_and_rows():
    from kvstreams import ops

    x, ids, t, grad = _case(6, 500, 8, torch.float32, 1)
    ids[0] = -1                       # a row without slots
    t[1] = -math.inf                  # the same, said by the values
    ids[2, 3:] = -1
    t[3, ::2] = -math.inf
    t[4, 1:] = -math.inf              # one slot left
    loss, lse, d = _check(x, ids, t, grad, 1.0, torch.float32)
    assert loss[0] == 0 and loss[1] == 0
    assert (d[:2] == 0).all()
    t[5] = math.nan                   # NaN: every slot empty
    loss, _ = ops.distill(x, ids, t)
    assert loss[5] == 0


def test_an_id_given_twice_adds_up():
    x, ids, t, grad = _case(4, 300, 6, torch.float32, 2)
    ids[:, 4] = ids[:, 1]
    ids[1] = ids[1, 0]
    _check(x, ids, t, grad, 1.0, torch.float32)


def test_masked_vocabulary():
    """Logits of -inf and of the type's lowest value, not named by the teacher, have probability 0
    and gradient 0; named by it with some weight, the loss is infinite."""
    from kvstreams import ops

    for low in (-math.inf, torch.finfo(torch.float32).min):
        x, ids, t, grad = _case(3, 700, 5, torch.float32, 3)
        free = torch.ones(3, 700, dtype=torch.bool, device="cuda").scatter_(1, ids, False)
        free[:, ::2] = False
        x[free] = low
        loss, lse, d = _check(x, ids, t, grad, 1.0, torch.float32)
        assert (d[free] == 0).all()
    x[0, ids[0, 0]] = -math.inf
    loss, _ = ops.distill(x, ids, t)
    assert loss[0] == math.inf and torch.isfinite(loss[1:]).all()
    x[1, 5] = math.nan
    assert ops.distill(x, ids, t)[0][1].isnan()


def test_whole_segments_masked():
    """Rows whose threads, batches or cluster segments see nothing but masked logits (one entry is
    left): lse is that entry, its probability 1.  A row of -inf only has no distribution: NaN."""
    from kvstreams import ops

    for vocab in (1000, 40000, 128256):
        for low in (-math.inf, torch.finfo(torch.float32).min):
            for at in (0, vocab // 2, vocab - 1):
                x = torch.full((2, vocab), low, device="cuda")
                x[:, at] = 3.0
                ids = torch.full((2, 1), at, dtype=torch.long, device="cuda")
                t = torch.zeros(2, 1, device="cuda")
                loss, lse = ops.distill(x, ids, t)
                assert (lse == 3.0).all() and (loss == 0).all()
                d = ops.distill_backward(x, ids, t, lse, torch.ones(2, device="cuda"))
                assert (d == 0).all()  # q = p = 1 there, 0 elsewhere
        x[0] = -math.inf
        loss, lse = ops.distill(x, ids, t)
        assert loss[0].isnan() and lse[0] == -math.inf and loss[1] == 0


def test_id_past_the_vocabulary_gives_nan():
    from kvstreams import ops

    x, ids, t, grad = _case(3, 100, 4, torch.float32, 4)
    ids[1, 2] = 100
    ids[2, 3] = 1 << 40
    loss, lse = ops.distill(x, ids, t)
    d = ops.distill_backward(x, ids, t, lse, grad)
    assert torch.isfinite(loss[0]) and loss[1:].isnan().all()
    assert torch.isfinite(d[0]).all() and d[1:].isnan().all()


def test_in_place_and_strided_rows():
    from kvstreams import ops

    x, ids, t, grad = _case(7, 333, 9, torch.float32, 5)
    wide = torch.full((7, 400), 7.0, device="cuda")
    wide[:, 3:336] = x
    view = wide[:, 3:336]
    # where a row's 16-byte loads begin decides the order of its sum, so the strided rows' loss
    # is held to the float64 bound, not to the packed rows' bits; the gradient is elementwise
    _check(view, ids, t, grad, 1.0, torch.float32)
    loss, lse = ops.distill(x, ids, t)
    want = ops.distill_backward(x, ids, t, lse, grad)
    assert torch.equal(ops.distill_backward(view, ids, t, lse, grad), want)
    got = ops.distill_backward(view, ids, t, lse, grad, out=view)
    assert got is view and torch.equal(view, want)
    assert (wide[:, :3] == 7).all() and (wide[:, 336:] == 7).all()
