"""The differentiable products keep pre-activations only where a backward can follow: not under
``torch.no_grad()`` or inference mode, whose operands are parameters that require gradients all the same
(every rollout, prefill and replay without gradients)."""

import contextlib

import pytest
import torch


@pytest.fixture
def calls(monkeypatch):
    """The launches of kvstreams.functional, on host tensors: what they were asked to keep."""
    from kvstreams import functional as KF

    seen = []

    def product(x, *weights, pre=None, activation=None, **kw):
        seen.append(pre)
        return x.new_zeros(x.shape[:-1] + (weights[0].shape[0],))

    monkeypatch.setattr(KF.ops, "linear", product)
    monkeypatch.setattr(KF.ops, "gated_linear", product)
    return seen


def _modes():
    return [("recording", contextlib.nullcontext, True), ("no_grad", torch.no_grad, False),
            ("inference", torch.inference_mode, False)]


@pytest.mark.parametrize("name,mode,kept", _modes())
@pytest.mark.parametrize("trainable", [True, False])
def test_pre_activations_are_kept_for_a_backward_only(calls, name, mode, kept, trainable):
    from kvstreams import functional as KF

    w, u = (torch.nn.Parameter(torch.zeros(48, 64), requires_grad=trainable) for _ in range(2))
    x = torch.zeros(5, 64)
    with mode():
        KF.gated_linear(x, w, u)
        KF.linear(x, w, activation="gelu")
        KF.linear(x, w)
    want = kept and trainable
    gated, act, plain = calls
    assert plain is None
    assert (gated is not None) == want and (act is not None) == want
    if want:
        assert gated.shape == (5, 96) and gated.dtype == torch.float32 and act.shape == (5, 48)


@pytest.mark.gpu
def test_memory_and_gradients_on_the_gpu():
    """Without gradients the call takes no more memory than the plain launch; with them the gradients
    are those of the plain launches."""
    from kvstreams import functional as KF, ops

    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(512, 256, generator=g, device="cuda").bfloat16()
    w, u = (torch.nn.Parameter(torch.randn(1024, 256, generator=g, device="cuda").bfloat16()) for _ in range(2))

    def peak(f):
        f(x, w, u)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        f(x, w, u)
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated() - before

    with torch.no_grad():
        assert peak(KF.gated_linear) == peak(ops.gated_linear) <= 2 * 512 * 1024 * 2
    gy = torch.randn(512, 1024, generator=g, device="cuda").bfloat16()
    KF.gated_linear(x, w, u).backward(gy)
    pre = ops.pre_buffer(x, 2048)
    ops.gated_linear(x, w.detach(), u.detach(), pre=pre)
    _, dw, du = ops.gated_linear_backward(gy, x, w.detach(), u.detach(), pre)
    assert torch.equal(w.grad, dw) and torch.equal(u.grad, du)
