"""Differentiable forms of the operators over wide rows of logits (a vocabulary, a large class set), for modules and losses in an autograd graph:

| here | kernels |
|---|---|
| ``token_logprobs``         | ``ag_token_logprobs`` + ``ag_token_logprobs_bwd`` |
| ``loss_topk_distillation`` | ``ag_topk_distill`` + ``ag_topk_distill_bwd`` |

The reference distils its surrogate from the classifier's full probability vector (models/shapley.py:96-106: ``models.shapley.
loss_logits_kl_divergence`` here).  These do the same for rows too wide for that: the teacher is recorded once as its top log-probabilities
(``token_logprobs(..., top_k)``) and the student is trained against the record (``loss_topk_distillation``).

Logits are fp32 or bf16 [..., V] on an MI355X; there is no CPU fallback.  Forward and backward read the logits once each and keep a few numbers
per row between them, so the logits must not be changed in place in the meantime (autograd checks that).  Loops that compute their own gradients
call ``ops.topk_distill``, which returns loss and gradient from one call.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from .. import ops


class Logprobs(NamedTuple):
    logp: Optional[Tensor]
    entropy: Tensor
    lse: Tensor
    top_ids: Optional[Tensor]
    top_logp: Optional[Tensor]


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top_k, temperature):
        r = ops.token_logprobs(logits, tokens, top_k, temperature)
        ctx.save_for_backward(logits, tokens, r.stats, r.top_ids)
        ctx.temperature = r.temperature
        ctx.set_materialize_grads(False)
        if r.top_ids is not None:
            ctx.mark_non_differentiable(r.top_ids)
        return r.logp, r.entropy, r.lse, r.top_ids, r.top_logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logp, g_entropy, g_lse, _g_ids, g_top):
        if g_logp is None and g_entropy is None and g_lse is None and g_top is None:
            return None, None, None, None
        logits, tokens, stats, top_ids = ctx.saved_tensors
        fwd = ops.TokenLogprobs(None, None, None, top_ids, None, stats, ctx.temperature)
        return ops.token_logprobs_bwd(logits, fwd, tokens, g_logp, g_entropy, g_lse, g_top), None, None, None


def token_logprobs(logits: Tensor, tokens: Optional[Tensor] = None, top_k: int = 0, temperature: float = 1.0) -> Logprobs:
    """``ops.token_logprobs`` on logits [..., V] and tokens [...] int64; every output but the ids is differentiable with respect to the logits."""
    lead, v = logits.shape[:-1], logits.shape[-1]
    logp, entropy, lse, ids, top = _TokenLogprobs.apply(logits.reshape(-1, v), None if tokens is None else tokens.reshape(-1), top_k, temperature)
    return Logprobs(None if logp is None else logp.view(lead), entropy.view(lead), lse.view(lead), None if ids is None else ids.view(*lead, top_k),
                    None if top is None else top.view(*lead, top_k))


class _TopkDistill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_ids, teacher_logp, weights, temperature, tail):
        r = ops.topk_distill(logits, teacher_ids, teacher_logp, weights, temperature, tail, want_grad=False)
        ctx.save_for_backward(logits, teacher_ids, teacher_logp, weights, r.stats)
        ctx.temperature, ctx.tail = temperature, tail
        ctx.set_materialize_grads(False)
        return r.loss.reshape(()), r.row_loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, g_row):
        if g_loss is None and g_row is None:
            return None, None, None, None, None, None
        logits, ids, tlp, weights, stats = ctx.saved_tensors
        d = ops.topk_distill_bwd(logits, ops.TopkDistill(None, None, None, stats), ids, tlp, weights, ctx.temperature, ctx.tail,
                                 d_loss=None if g_loss is None else g_loss.reshape(1), d_row_loss=g_row)
        return d, None, None, None, None, None


def loss_topk_distillation(logits: Tensor, teacher_ids: Tensor, teacher_logp: Tensor, weights: Optional[Tensor] = None, temperature: float = 1.0,
                           tail: bool = False) -> Tuple[Tensor, Tensor]:
    """``ops.topk_distill`` on logits [..., V], teacher_ids / teacher_logp [..., K] and weights [...] -> (loss, row losses [...]), both
    differentiable with respect to the logits (the teacher's record and the weights get no gradient)."""
    lead, v, k = logits.shape[:-1], logits.shape[-1], teacher_ids.shape[-1]
    loss, row = _TopkDistill.apply(logits.reshape(-1, v), teacher_ids.reshape(-1, k), teacher_logp.detach().reshape(-1, k),
                                   None if weights is None else weights.detach().reshape(-1), temperature, tail)
    return loss, row.view(lead)
