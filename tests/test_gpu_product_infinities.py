"""Infinities and NaN through the products, entry by entry: forward, gated and both gradients, in every kernel
(3 rows: weights streamed; 300: pairs of CTAs; 600 x 1500 x 14344: cut tiles).  What they do not touch keeps its bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = [(3, 200, 256), (300, 200, 256), (300, 201, 256), (600, 1500, 14344)]


def _rand(seed, *shape, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).bfloat16()


def _planted(rows, k):
    x = _rand(1, rows, k)
    bad = x.clone()
    bad[1, 5] = math.nan
    bad[2, 7] = math.inf
    return x, bad, [i for i in range(rows) if i not in (1, 2)]


def _weights(seed, n, k):
    w = _rand(seed, n, k, scale=0.05)
    w[4, 7] = 0  # 0 times infinity
    return w


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("rows,n,k", SIZES)
def test_forward(rows, n, k, act):
    from kvstreams import ops

    x, bad, keep = _planted(rows, k)
    w = _weights(2, n, k)
    clean, y = ops.linear(x, w, activation=act), ops.linear(bad, w, activation=act)
    assert torch.equal(y[keep], clean[keep])
    assert y[1].isnan().all()
    up, down, none = w[:, 7] > 0, w[:, 7] < 0, w[:, 7] == 0
    assert none[4] and y[2][none].isnan().all()
    assert (y[2][up] == math.inf).all()
    low = y[2][down]
    if act is None:
        assert (low == -math.inf).all()
    elif act == "relu":
        assert (low == 0).all()
    else:  # -inf times 0
        assert (low.isnan() | (low == 0)).all()


@pytest.mark.parametrize("rows,n,k", SIZES)
def test_gated(rows, n, k):
    from kvstreams import ops

    x, bad, keep = _planted(rows, k)
    w, u = _weights(2, n, k), _weights(3, n, k)
    pre = ops.pre_buffer(x, 2 * n)
    clean, h = ops.gated_linear(x, w, u), ops.gated_linear(bad, w, u, pre=pre)
    assert torch.equal(h[keep], clean[keep])
    assert h[1].isnan().all() and pre[1].isnan().all()
    gate, up = w[:, 7].float(), u[:, 7].float()
    for half, col in ((pre[2, :n], gate), (pre[2, n:], up)):
        assert torch.equal(half.nan_to_num(0.0, 1.0, -1.0), torch.sign(col))
    on = (gate > 0) & (up != 0)
    assert torch.equal(h[2][on].float(), torch.sign(up[on]) * math.inf)
    assert h[2][(gate == 0) | (up == 0)].isnan().all()
    assert h[2][(gate < 0) & (up != 0)].isnan().all()  # silu(-inf), 0 or nan, times infinity


@pytest.mark.parametrize("rows,n,k", SIZES)
def test_gradients(rows, n, k):
    from kvstreams import ops

    x, bad, keep = _planted(rows, k)
    w, gy = _weights(2, n, k), _rand(4, rows, n)
    dx, dw, db = ops.linear_backward(gy, x, w, bias_grad=True)
    # infinities in x: their columns of dW, and nothing else
    bx, bw, bb = ops.linear_backward(gy, bad, w, bias_grad=True)
    cols = [c for c in range(k) if c not in (5, 7)]
    assert torch.equal(bx, dx) and torch.equal(bb, db) and torch.equal(bw[:, cols], dw[:, cols])
    assert bw[:, 5].isnan().all()
    some = gy[2] != 0
    assert torch.equal(bw[some, 7].float(), torch.sign(gy[2][some].float()) * math.inf)
    # in gy: their rows of dx, their outputs' rows of dW and entries of db
    bg = gy.clone()
    bg[1, 9] = math.nan
    bg[2, 11] = -math.inf
    bx, bw, bb = ops.linear_backward(bg, x, w, bias_grad=True)
    outs = [c for c in range(n) if c not in (9, 11)]
    assert torch.equal(bx[keep], dx[keep]) and torch.equal(bw[outs], dw[outs]) and torch.equal(bb[outs], db[outs])
    assert bx[1].isnan().all() and bw[9].isnan().all() and bb[9].isnan() and bb[11] == -math.inf
    some = w[11] != 0
    assert torch.equal(bx[2][some].float(), -torch.sign(w[11][some].float()) * math.inf)
    some = x[2] != 0
    assert torch.equal(bw[11][some].float(), -torch.sign(x[2][some].float()) * math.inf)


@pytest.mark.parametrize("rows,n,k", SIZES[:3])
def test_gated_gradients(rows, n, k):
    from kvstreams import ops

    x, _, keep = _planted(rows, k)
    w, u, gh = _weights(2, n, k), _weights(3, n, k), _rand(4, rows, n)
    pre = ops.pre_buffer(x, 2 * n)
    ops.gated_linear(x, w, u, pre=pre)
    dx, dw, du = ops.gated_linear_backward(gh, x, w, u, pre)
    bg = gh.clone()
    bg[1, 9] = math.nan
    bg[2, 11] = math.inf
    bx, bw, bu = ops.gated_linear_backward(bg, x, w, u, pre)
    outs = [c for c in range(n) if c not in (9, 11)]
    assert torch.equal(bx[keep], dx[keep]) and torch.equal(bw[outs], dw[outs]) and torch.equal(bu[outs], du[outs])
    assert bx[1].isnan().all() and bw[9].isnan().all() and bu[9].isnan().all()
    assert not torch.isfinite(bx[2]).any() and not torch.isfinite(bu[11]).any()
