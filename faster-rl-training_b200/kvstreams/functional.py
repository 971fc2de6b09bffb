"""Differentiable forms of the library's products and of the distillation loss.

:func:`linear` and :func:`gated_linear` are the projections of a decoder layer (model.py:58-63,
74-86 of the reference) with bias, activation, gate product and residual in the product's own
launch; :func:`distill` is the loss of logits rows against a teacher's top logits.  Each is one
autograd node over the pair of kernels in :mod:`kvstreams.ops`; only the gradients that are
needed are computed, and what an activation's gradient needs is kept in float32, where autograd
records: a node's ``needs_input_grad`` is true for a parameter under ``torch.no_grad()`` too, so the
mode is asked before the node (whose forward always runs with recording off).

Capturing a backward pass into a CUDA graph: PyTorch ties the accumulation into a leaf to the stream
of the leaf's first use, so release every eager graph over the same leaves before the capture (or
capture :func:`kvstreams.ops.linear_backward` and its like, which are plain launches).
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops

__all__ = ["distill", "gated_linear", "linear", "product_kernels"]


def product_kernels(x: torch.Tensor, *weights: torch.Tensor) -> bool:
    """Whether :func:`linear` / :func:`gated_linear` take these operands: bf16/fp16 CUDA tensors of
    one type, inner sizes that are multiples of 8."""
    return (x.is_cuda and x.dtype in (torch.bfloat16, torch.float16)
            and all(w.is_cuda and w.dtype == x.dtype and w.shape[1] % 8 == 0 for w in weights))


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, recorded):
        pre = None
        if recorded and activation is not None and any(ctx.needs_input_grad[:3]):
            pre = ops.pre_buffer(x, weight.shape[0])
        y = ops.linear(x, weight, bias=bias, residual=residual, activation=activation, pre=pre)
        ctx.save_for_backward(x, weight, pre)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, weight, pre = ctx.saved_tensors
        nx, nw, nb, nr = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if nx or nw or nb:
            dx, dw, db = ops.linear_backward(gy, x, weight, pre=pre, activation=ctx.activation, bias_grad=nb,
                                             need_dx=nx, need_dw=nw)
        return dx, dw, db, gy if nr else None, None, None


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, activation, recorded):
        pre = ops.pre_buffer(x, 2 * w_gate.shape[0]) if recorded and any(ctx.needs_input_grad[:3]) else None
        h = ops.gated_linear(x, w_gate, w_up, activation=activation, pre=pre)
        ctx.save_for_backward(x, w_gate, w_up, pre)
        ctx.activation = activation
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, gh):
        x, w_gate, w_up, pre = ctx.saved_tensors
        nx, ng, nu = ctx.needs_input_grad[:3]
        dx, dg, du = ops.gated_linear_backward(gh, x, w_gate, w_up, pre, activation=ctx.activation, need_dx=nx,
                                               need_dw=ng or nu)
        return dx, dg if ng else None, du if nu else None, None, None


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, temperature):
        loss, lse = ops.distill(logits, ids, teacher, temperature)
        ctx.save_for_backward(logits, ids, teacher, lse)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, ids, teacher, lse = ctx.saved_tensors
        return ops.distill_backward(logits, ids, teacher, lse, g, ctx.temperature), None, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           residual: Optional[torch.Tensor] = None, activation: Optional[str] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` (:func:`kvstreams.ops.linear`), differentiable in x,
    weight, bias and residual."""
    return _Linear.apply(x, weight, bias, residual, activation, torch.is_grad_enabled())


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                 activation: Optional[str] = "silu") -> torch.Tensor:
    """``act(x @ w_gate.T) * (x @ w_up.T)`` (:func:`kvstreams.ops.gated_linear`), differentiable in x
    and both weights."""
    return _GatedLinear.apply(x, w_gate, w_up, activation, torch.is_grad_enabled())


def distill(logits: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """Per-row loss of ``logits`` ``[rows, vocab]`` against a teacher's top logits
    (:func:`kvstreams.ops.distill`), differentiable in the logits."""
    return _Distill.apply(logits, ids, teacher, float(temperature))
