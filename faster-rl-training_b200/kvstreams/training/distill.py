"""Distillation of replayed rollouts from a teacher's top logits.

The trainer replays a batch exactly as for :func:`token_logprobs` (training/logprobs.py:10-25 of the
reference: masked forward, lm_head, log-softmax), and compares each position's distribution with the
``k`` best logits that a teacher gave there, instead of with the one token that was sampled.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import ops
from ..functional import product_kernels
from .logprobs import _CHUNK_TOKENS
from .replay import Batch


def _wide_logits(model, h: torch.Tensor) -> torch.Tensor:
    logits = model.logits(h)
    return logits.float() if logits.dtype in (torch.bfloat16, torch.float16) else logits


class _LmHeadDistill(torch.autograd.Function):
    """One chunk of lm_head -> distillation loss.  Only the hidden states and each row's log-sum-exp
    are kept; the backward recomputes the chunk's logits, turns them into their gradient in the
    weight's type (in place when that is the logits' own) and runs the two products of dh and dW."""

    @staticmethod
    def forward(ctx, h, weight, ids, teacher, temperature, model):
        loss, lse = ops.distill(_wide_logits(model, h), ids, teacher, temperature)
        ctx.save_for_backward(h, weight, ids, teacher, lse)
        ctx.temperature, ctx.model = temperature, model
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        h, weight, ids, teacher, lse = ctx.saved_tensors
        logits = _wide_logits(ctx.model, h)
        same = weight.dtype == logits.dtype
        dlog = ops.distill_backward(logits, ids, teacher, lse, g, ctx.temperature,
                                    out_dtype=weight.dtype, out=logits if same else None)
        del logits
        nh, nw = ctx.needs_input_grad[:2]
        if product_kernels(h, weight):
            dh, dw, _ = ops.linear_backward(dlog, h, weight, need_dx=nh, need_dw=nw)
        else:
            dh = dlog @ weight if nh else None
            dw = dlog.t() @ h.to(weight.dtype) if nw else None
        return dh, dw, None, None, None, None


def distill_loss(model, batch: Batch, ids: torch.Tensor, teacher: torch.Tensor,
                 temperature: float = 1.0) -> torch.Tensor:
    """``[B, T]`` loss of the replayed student at every position against the teacher's top logits.

    ``ids`` / ``teacher`` ``[B, T, k]``: the teacher's best entries and their logits for token ``t``
    given the context of ``t - 1`` (the alignment of :func:`token_logprobs`; position 0 is 0 and its
    slots are not read).  A slot with a negative id or a teacher value of -inf is empty; a position
    without slots (padding, prompt) has loss 0.  Differentiable in the model's parameters; lm_head and
    loss run in token chunks, so the ``[B, T, V]`` logits never exist at once."""
    dev = model.device
    tokens = batch.tokens.to(dev)
    B, T = tokens.shape
    if ids.shape != teacher.shape or tuple(ids.shape[:2]) != (B, T) or ids.dim() != 3:
        raise ValueError(f"ids and teacher must be [{B}, {T}, k] (got {tuple(ids.shape)} and {tuple(teacher.shape)})")
    hidden = model.forward_hidden(tokens, batch.positions.to(dev), batch.mask.to(dev))
    flat_h = hidden[:, :-1].reshape(-1, hidden.shape[-1])
    flat_i = ids.to(dev)[:, 1:].reshape(-1, ids.shape[-1])
    flat_t = teacher.to(dev)[:, 1:].reshape(-1, ids.shape[-1])
    parts = [_LmHeadDistill.apply(flat_h[a:a + _CHUNK_TOKENS], model.lm_head.weight, flat_i[a:a + _CHUNK_TOKENS],
                                  flat_t[a:a + _CHUNK_TOKENS], float(temperature), model)
             for a in range(0, flat_h.shape[0], _CHUNK_TOKENS)]
    want = torch.float64 if hidden.dtype == torch.float64 else torch.float32
    res = torch.cat(parts) if parts else torch.empty(0, dtype=want, device=dev)
    return torch.cat([torch.zeros(B, 1, dtype=res.dtype, device=dev), res.view(B, T - 1)], dim=1)


@torch.no_grad()
def top_logits(model, batch: Batch, k: int):
    """``(ids, logits)`` ``[B, T, k]`` of ``model`` as a teacher over a replayed batch, aligned for
    :func:`distill_loss`; position 0 and padded positions have empty slots (id -1, logit -inf)."""
    dev = model.device
    tokens = batch.tokens.to(dev)
    B, T = tokens.shape
    hidden = model.forward_hidden(tokens, batch.positions.to(dev), batch.mask.to(dev))
    flat = hidden[:, :-1].reshape(-1, hidden.shape[-1])
    wide = torch.float64 if hidden.dtype == torch.float64 else torch.float32
    ids = torch.full((B, T, k), -1, dtype=torch.long, device=dev)
    top = torch.full((B, T, k), float("-inf"), dtype=wide, device=dev)
    for a in range(0, flat.shape[0], _CHUNK_TOKENS):
        v, i = _wide_logits(model, flat[a:a + _CHUNK_TOKENS]).topk(k, dim=-1)
        at = torch.arange(a, a + v.shape[0], device=dev)
        ids[at // (T - 1), at % (T - 1) + 1] = i
        top[at // (T - 1), at % (T - 1) + 1] = v
    pad = torch.arange(T, device=dev)[None, :] >= batch.lengths.to(dev)[:, None]
    ids[pad] = -1
    top[pad] = float("-inf")
    return ids, top
