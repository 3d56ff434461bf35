"""Learning from a teacher's most likely tokens.

``token_logprobs(teacher_logits, ..., top_k=k)`` leaves the full-precision model's best tokens and their log
probabilities, a few numbers a token that can be stored; ``distillation_loss`` compares a student's logits with them,
in one pass over the logits, and is differentiable in them.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from . import kernels as K
from .scoring import logit_rows, row_values


class Distillation(NamedTuple):
    """``loss`` fp32 ``[...]``; ``stats`` fp32 ``[..., 8]`` for the backward pass."""
    loss: torch.Tensor
    stats: torch.Tensor


def _checked(logits, ids, teacher, temperature, tail):
    z, N, V, lead = logit_rows(logits)
    if not isinstance(ids, torch.Tensor) or ids.dtype is not torch.int64 or ids.dim() != len(lead) + 1 or ids.shape[:-1] != lead \
            or ids.get_device() != logits.get_device():
        raise ValueError(f"teacher_ids must be int64 {[*lead, 'k']} on {logits.device}")
    k = ids.shape[-1]
    if not 1 <= k <= nat.RQ_DISTILL_MAX_TOP:
        raise ValueError(f"the teacher's list must hold 1 to {nat.RQ_DISTILL_MAX_TOP} tokens, got {k}")
    teacher = row_values(teacher, ids.shape, logits, "teacher_logprobs")
    if teacher.requires_grad and torch.is_grad_enabled():
        raise ValueError("teacher_logprobs are constants and would get no gradient; detach them")
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature must be 1e-6 to 1e6, got {temperature}")
    if tail not in nat.TAILS:
        raise ValueError(f"tail must be one of {sorted(nat.TAILS)}, got {tail!r}")
    if tail == "bucket" and temperature != 1.0:
        raise ValueError("tail='bucket' takes the teacher's probabilities as they are: temperature must be 1")
    return z, ids if ids.is_contiguous() else ids.contiguous(), teacher, N, V, k, temperature, nat.TAILS[tail], lead


def _forward(logits, ids, teacher, temperature, tail):
    z, ids, teacher, N, V, k, temperature, tail, lead = _checked(logits, ids, teacher, temperature, tail)
    return Distillation(*K.distill_loss(z, ids, teacher, N, V, k, temperature, tail, lead))


def _backward(logits, ids, teacher, stats, grad_loss, temperature, tail):
    z, ids, teacher, N, V, k, temperature, tail, lead = _checked(logits, ids, teacher, temperature, tail)
    grad_loss = row_values(grad_loss, lead, logits, "grad_loss")
    stats = row_values(stats, (*lead, nat.RQ_DISTILL_STATS), logits, "stats (distillation_loss')")
    return K.distill_loss_grad(z, ids, teacher, N, V, k, temperature, tail, stats, grad_loss, lead)


class _DistillationLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, temperature, tail):
        r = _forward(logits, ids, teacher, temperature, tail)
        nat.save_for_backward(ctx, logits, ids, teacher, r.stats)
        ctx.how = temperature, tail
        ctx.mark_non_differentiable(r.stats)
        ctx.set_materialize_grads(False)                 # or backward gets zeros of the statistics' size
        return tuple(r)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, _):
        if grad_loss is None:
            return None, None, None, None, None
        logits, ids, teacher, stats = nat.saved_for_backward(ctx)
        return _backward(logits, ids, teacher, stats, grad_loss, *ctx.how), None, None, None, None


def distillation_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, temperature: float = 1.0,
                      tail: str = "renormalise") -> Distillation:
    """The Kullback-Leibler divergence from a teacher's top tokens to ``softmax(logits / temperature)``, one value a row:
    logits [..., V] (fp16, bf16 or fp32), ``teacher_ids`` (int64) and ``teacher_logprobs`` (fp32) [..., k], k up to 256, in any
    order, as ``token_logprobs``' ``top_ids`` and ``top_logprobs`` are; an id below 0 is no entry.

    ``tail="renormalise"``: the teacher's distribution is ``softmax(teacher_logprobs / temperature)`` over its list.
    ``tail="bucket"`` (temperature 1): it is ``exp(teacher_logprobs)``, and what is left of 1 is compared with the student's
    probability of all other tokens, as one class.  The loss is not multiplied by ``temperature ** 2``.

    Masked logits have probability 0: an unlisted one counts for nothing, a listed one that the teacher gives
    a probability makes the loss inf.  A row without entries has loss 0 and no gradient; a row with nothing but -inf has
    loss inf (0 without a teacher's probability) and no gradient; a NaN, a logit of +inf or an id outside the vocabulary makes
    its row NaN.  The teacher's side is constant; forward-mode tangents are refused."""
    nat.refuse_tangents("distillation_loss", logits, teacher_logprobs)
    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        _checked(logits, teacher_ids, teacher_logprobs, temperature, tail)         # under autograd; forward runs without
        return Distillation(*_DistillationLoss.apply(logits, teacher_ids, teacher_logprobs, temperature, tail))
    return _forward(logits, teacher_ids, teacher_logprobs, temperature, tail)


class _DistillationLossGrad(torch.autograd.Function):
    """The gradient from inputs that require grad: no constant, so a derivative of it is refused."""
    @staticmethod
    def forward(ctx, *args):
        return _backward(*args)

    @staticmethod
    def backward(ctx, _):
        raise NotImplementedError("distillation_loss_backward has no backward pass: call it under torch.no_grad() or on "
                                  "detached tensors")


def distillation_loss_backward(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor,
                               stats: torch.Tensor, grad_loss: torch.Tensor, temperature: float = 1.0,
                               tail: str = "renormalise") -> torch.Tensor:
    """The gradient of ``logits`` from the gradient of ``loss``, in the logits' dtype; ``stats`` is what ``distillation_loss``
    returned for the same arguments.  It cannot be differentiated further."""
    nat.refuse_tangents("distillation_loss_backward", logits, teacher_logprobs, stats, grad_loss)
    args = logits, teacher_ids, teacher_logprobs, stats, grad_loss, temperature, tail
    if torch.is_grad_enabled() and (getattr(logits, "requires_grad", False) or getattr(stats, "requires_grad", False) or
                                    getattr(grad_loss, "requires_grad", False)):
        _checked(logits, teacher_ids, teacher_logprobs, temperature, tail)
        return _DistillationLossGrad.apply(*args)
    return _backward(*args)
