"""The products and the distillation loss run together: a replayed batch through a model whose
layers use them (TinyLM.fused_products), the loss against a teacher's top logits, and the gradients
of every parameter -- against float64 and against differences."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

CFG = dict(vocab_size=333, d_model=64, n_layers=2, n_heads=4, n_kv_heads=2, d_ff=136)


def _model(dtype, seed=0, **kw):
    from kvstreams.config import ModelConfig
    from kvstreams.model import TinyLM

    torch.manual_seed(seed)
    return TinyLM(ModelConfig(**{**CFG, "init_std": 0.1, **kw})).cuda().to(dtype)


def _batch(B=3, T=40, seed=0, vocab=333):
    from kvstreams.training import Batch

    g = torch.Generator().manual_seed(seed)
    lengths = torch.tensor([T, T - 7, 1])[:B]
    ev = torch.full((B, T), (1 << 63) - 1, dtype=torch.long)
    ev[0, 3:9] = 20
    ev[1, 1:5] = 11
    return Batch(torch.randint(0, vocab, (B, T), generator=g), torch.arange(T).expand(B, T).contiguous(), ev.cuda(),
                 torch.ones(B, T, dtype=torch.bool), torch.zeros(B, T, dtype=torch.float64), lengths)


def _teacher(batch, k=12):
    from kvstreams.training import top_logits

    ids, top = top_logits(_model(torch.float64, seed=7), batch, k)
    ids[0, 5, 4:] = -1  # fewer slots
    ids[0, 6] = -1      # none
    return ids, top


def test_float64_gradients_match_differences():
    """float64 model: the loss equals the definition, and its gradient along random directions
    equals central differences (h = 1e-4: truncation h^2 / 6 |f'''| ~ 1e-8, rounding eps |f| / h ~ 1e-11)."""
    from kvstreams.training import distill_loss

    model, batch = _model(torch.float64), _batch()
    ids, top = _teacher(batch)
    T = 1.3
    loss = distill_loss(model, batch, ids, top, T)
    logits = model(batch.tokens.cuda(), batch.positions.cuda(), batch.mask).detach()
    kept = (ids >= 0) & (top > -np.inf)
    lp = torch.log_softmax(torch.where(kept, top / T, -1e300), -1)
    logq = torch.log_softmax(logits / T, -1)
    shifted = torch.cat([logq[:, :1], logq[:, :-1]], 1).gather(2, ids.clamp(min=0))
    want = torch.where(kept, lp.exp() * (lp - shifted), 0.0).sum(-1)
    want[:, 0] = 0
    assert (loss - want).abs().max().item() <= 1e-11
    assert (loss[2] == 0).all() and loss[0, 6] == 0
    w = torch.rand(loss.shape, dtype=torch.float64, device="cuda")
    (loss * w).sum().backward()
    for seed in range(3):
        torch.manual_seed(100 + seed)
        dirs = [torch.randn_like(p) for p in model.parameters()]
        slope = sum((p.grad * d).sum() for p, d in zip(model.parameters(), dirs)).item()
        vals = []
        for h in (1e-4, -1e-4):
            with torch.no_grad():
                for p, d in zip(model.parameters(), dirs):
                    p.add_(d, alpha=h)
                vals.append((distill_loss(model, batch, ids, top, T) * w).sum().item())
                for p, d in zip(model.parameters(), dirs):
                    p.sub_(d, alpha=h)
        diff = (vals[0] - vals[1]) / 2e-4
        assert abs(diff - slope) <= 1e-4 * max(1.0, abs(slope)), (diff, slope)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_half_step_matches_float64(dtype):
    """A half-precision training step with the products against the same weights in float64.  Each
    tensor between kernels carries half a step, eps / 2, and passes about twenty of them; the
    gradients are compared as whole tensors, whose random roundings add as squares: 10 eps / 2 in
    norm is over twice sqrt(20) eps / 2.  The default (PyTorch) products round the same tensors,
    and one more (gate|up), so the products may not be further off than 1.5 times them."""
    from kvstreams.training import distill_loss

    batch = _batch(T=70)
    ids, top = _teacher(batch)
    ref = _model(torch.float64)
    model = _model(dtype)
    with torch.no_grad():
        for p, q in zip(ref.parameters(), model.parameters()):
            p.copy_(q.double())
    assert not model.fused_products
    errs = {}
    w = torch.rand(batch.tokens.shape, device="cuda")
    (distill_loss(ref, batch, ids, top) * w).sum().backward()
    for fused in (False, True):
        model.fused_products = fused
        assert model.fused_products is fused
        model.zero_grad()
        loss = distill_loss(model, batch, ids, top)
        (loss * w).sum().backward()
        errs[fused] = {n: ((p.grad.double() - q.grad).norm() / q.grad.norm()).item()
                       for (n, p), q in zip(model.named_parameters(), ref.parameters())}
    half = torch.finfo(dtype).eps / 2
    for n, e in errs[True].items():
        assert e <= 10 * half, (n, e / half)
        assert e <= max(1.5 * errs[False][n], 4 * half), (n, e / half, errs[False][n] / half)


def test_fused_products_leave_other_models_alone():
    """float32 models keep their results to the bit; half models keep theirs while it is off."""
    for dtype in (torch.float32, torch.bfloat16):
        model, batch = _model(dtype), _batch()
        args = (batch.tokens.cuda(), batch.positions.cuda(), batch.mask)
        with torch.no_grad():
            before = model(*args)
            model.fused_products = True
            during = model(*args)
            model.fused_products = False
            after = model(*args)
        assert torch.equal(before, after)
        if dtype == torch.float32:
            assert torch.equal(before, during)
        else:
            assert not torch.equal(before, during)  # the products did run


def test_cached_decode_with_the_products():
    """Prefill and single-token decode of a bf16 model through the paged cache with the products
    agree with the same model without them (the same roundings but one; logits of size ~1)."""
    from kvstreams.paged_cache import PagedKVCache

    model = _model(torch.bfloat16)
    outs = []
    for fused in (False, True):
        model.fused_products = fused
        cache = PagedKVCache(2, 2, 16, block_size=16, num_blocks=64, dtype=torch.bfloat16, max_seqs=4)
        for s in range(3):
            cache.add_sequence(s)
        g = torch.Generator().manual_seed(3)
        counts = [5, 17, 1]
        toks = torch.randint(0, 333, (sum(counts),), generator=g)
        pos = torch.cat([torch.arange(c) for c in counts])
        rows = [model.forward_cached_batch(toks, pos, cache, [0, 1, 2], counts)]
        for step in range(3):
            t = torch.randint(0, 333, (3,), generator=g)
            rows.append(model.forward_cached_batch(t, torch.tensor([c + step for c in counts]), cache, [0, 1, 2]))
        outs.append(torch.cat(rows))
    scale = outs[0].abs().max().item()
    assert (outs[0] - outs[1]).abs().max().item() <= 16 * 2 ** -8 * max(scale, 1.0)


def test_frozen_weights_and_missing_gradients():
    from kvstreams import functional as KF

    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(5, 64, generator=g, device="cuda").bfloat16()
    w, u = (torch.randn(48, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
    b = torch.randn(48, generator=g, device="cuda").bfloat16()
    for need in [(True, False, False), (False, True, False), (False, False, True), (True, True, True)]:
        xs, ws, bs = (t.clone().requires_grad_(n) for t, n in zip((x, w, b), need))
        KF.linear(xs, ws, bs, activation="gelu").sum().backward()  # (an expanded upstream gradient)
        assert [t.grad is not None for t in (xs, ws, bs)] == list(need)
        xs, ws, us = (t.clone().requires_grad_(n) for t, n in zip((x, w, u), need))
        KF.gated_linear(xs, ws, us).sum().backward()
        assert [t.grad is not None for t in (xs, ws, us)] == list(need)
    r = torch.randn(5, 48, generator=g, device="cuda").bfloat16().requires_grad_()
    KF.linear(x, w, residual=r).backward(torch.ones(5, 48, device="cuda").bfloat16())
    assert (r.grad == 1).all()
    # shared weights: the gradients of both uses add up
    ws = w.clone().requires_grad_()
    y = KF.linear(x, ws) + KF.linear(x, ws)
    y.sum().backward()
    one = w.clone().requires_grad_()
    KF.linear(x, one).sum().backward()
    assert torch.equal(ws.grad, one.grad * 2)
