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

Forward and backward can be captured into a HIP graph: warm up on a side stream, let no eager graph of the same leaves live on, and take the
gradient with ``torch.autograd.grad`` (torch ends the process where a captured ``backward`` meets the accumulator of an eager one).
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
        r = ops._token_logprobs(logits, tokens, top_k, temperature, no_views=True)
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


def _lead(who: str, logits: Tensor) -> torch.Size:
    if logits.dim() == 0:
        raise ValueError(f"{who}: logits must be [..., vocabulary]; got a number")
    return logits.shape[:-1]


def _rows(who: str, name: str, t: Optional[Tensor], lead: torch.Size, dims: int) -> Optional[Tensor]:
    """``t`` [*lead, any] (``dims`` 2) or [*lead] (1) with its leading dimensions as one; as it is where it has that form already (a view would be a
    node of the autograd graph).  Other leading dimensions than the logits' are refused: [3, 2] numbers for [2, 3] rows are as many, not the same."""
    if t is None:
        return None
    own = t.shape[:t.dim() - dims + 1]
    if t.dim() == dims and own.numel() == lead.numel():
        return t
    if t.dim() < dims - 1 or own != lead:
        raise ValueError(f"{who}: {name} must be {[*lead, '...'] if dims == 2 else list(lead)}; got {list(t.shape)}")
    return t.reshape(lead.numel(), t.shape[-1]) if dims == 2 else t.reshape(-1)


def _back(t: Optional[Tensor], lead) -> Optional[Tensor]:
    return t if t is None or len(lead) == 1 else t.view(lead + t.shape[1:])


def token_logprobs(logits: Tensor, tokens: Optional[Tensor] = None, top_k: int = 0, temperature: float = 1.0) -> Logprobs:
    """``ops.token_logprobs`` on logits [..., V] (a single row [V] among them: results without its dimension) and tokens [...] int64; every output
    but the ids is differentiable with respect to the logits."""
    who = "token_logprobs"
    lead = _lead(who, logits)
    out = _TokenLogprobs.apply(_rows(who, "logits", logits, lead, 2), _rows(who, "tokens", tokens, lead, 1), top_k, temperature)
    return Logprobs(*(_back(t, lead) for t in out))


class _TopkDistill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_ids, teacher_logp, weights, temperature, tail):
        r = ops._topk_distill(logits, teacher_ids, teacher_logp, weights, temperature, tail, want_grad=False, loss_shape=())
        ctx.save_for_backward(logits, teacher_ids, teacher_logp, weights, r.stats)
        ctx.temperature, ctx.tail = temperature, tail
        ctx.set_materialize_grads(False)
        return r.loss, r.row_loss

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
    who = "loss_topk_distillation"
    lead = _lead(who, logits)
    loss, row = _TopkDistill.apply(_rows(who, "logits", logits, lead, 2), _rows(who, "teacher_ids", teacher_ids, lead, 2),
                                   _rows(who, "teacher_logp", teacher_logp, lead, 2), _rows(who, "weights", weights, lead, 1), temperature, tail)
    return loss, _back(row, lead)
