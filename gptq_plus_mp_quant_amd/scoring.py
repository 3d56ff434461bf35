"""What a (quantised) model answers, from its logits: the log probability of given tokens, the entropy of
every distribution and the most likely alternatives, in one pass over the logits, and the gradient of
the logits.

Perplexity is ``(-token_logprobs(logits, targets).logprob).mean().exp()``; a static saliency or a refreshed
gradient starts from ``token_logprobs(...).logprob.sum().backward()``.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from . import kernels as K


class TokenLogprobs(NamedTuple):
    """``logprob`` and ``entropy`` fp32 ``[...]``; ``top_ids`` int64 and ``top_logprobs`` fp32
    ``[..., top_k]``, the most likely first; ``stats`` fp32 ``[..., 3]`` for the backward pass (the row's
    maximum, log sum exp(z - max), entropy)."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor
    stats: torch.Tensor


def _rows(logits, targets):
    """(logits [N, V] with unit column stride, targets [N], N, V, the leading dimensions)."""
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda):
        nat.require_gpu(logits, "logits")
    if logits.dtype not in nat.DTYPE_CODES:
        raise TypeError(f"logits: unsupported dtype {logits.dtype}; expected float16, bfloat16 or float32")
    shape = logits.shape
    if len(shape) < 1 or shape[-1] == 0:
        raise ValueError("logits must be [..., V] with V > 0")
    lead = shape[:-1]
    if not isinstance(targets, torch.Tensor) or targets.dtype is not torch.int64 or targets.shape != lead or \
            targets.get_device() != logits.get_device():
        raise ValueError(f"targets must be int64 {list(lead)} on {logits.device}")
    V = shape[-1]
    z = logits if len(shape) == 2 else logits.reshape(-1, V)
    s0, s1 = z.stride()
    if s1 != 1 or s0 < V:
        z = z.contiguous()
        if z.stride(0) < V:                      # one row: its stride is never used
            z = z.as_strided((z.shape[0], V), (V, 1))
    t = targets if targets.dim() == 1 else targets.reshape(-1)
    return z, t if t.is_contiguous() else t.contiguous(), z.shape[0], V, lead


def _forward(logits, targets, top_k, ignore_index):
    z, t, N, V, lead = _rows(logits, targets)
    top_k = int(top_k)
    if not 0 <= top_k <= min(nat.RQ_SCORE_MAX_TOP, V):
        raise ValueError(f"top_k must be 0 to {min(nat.RQ_SCORE_MAX_TOP, V)}, got {top_k}")
    return TokenLogprobs(*K.token_logprobs(z, t, N, V, top_k, int(ignore_index), lead))


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, ignore_index):
        r = _forward(logits, targets, top_k, ignore_index)
        ctx.save_for_backward(logits, targets, r.stats)
        ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(r.top_ids, r.top_logprobs, r.stats)
        return tuple(r)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_logprob, grad_entropy, *_):
        logits, targets, stats = ctx.saved_tensors
        return _backward(logits, targets, stats, grad_logprob, grad_entropy, ctx.ignore_index), None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_k: int = 0, ignore_index: int = -100) -> TokenLogprobs:
    """Score ``targets`` [...] (int64) under ``logits`` [..., V] (fp16, bf16 or fp32).

    ``logprob`` is 0 where the target is ``ignore_index`` and NaN for another target outside the vocabulary.
    ``top_k`` (0 to 64) alternatives are ordered by their logit, equal ones by their index.  Masked
    logits (-inf, or a large negative number) have probability 0; a row with nothing but -inf has
    logprob -inf, entropy 0 and no gradient; a row with a NaN or +inf is NaN.  ``logprob`` and
    ``entropy`` are differentiable in ``logits``, ``top_logprobs`` is not; forward-mode tangents are refused."""
    nat.refuse_tangents("token_logprobs", logits)
    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, top_k, ignore_index))
    return _forward(logits, targets, top_k, ignore_index)


def _row_values(g, lead, like, name):
    """A float32 tensor of the given shape on like's device, contiguous."""
    if not isinstance(g, torch.Tensor) or g.dtype is not torch.float32 or g.shape != lead or \
            g.get_device() != like.get_device():
        raise ValueError(f"{name} must be float32 {list(lead)} on {like.device}")
    return g if g.is_contiguous() else g.contiguous()


class _TokenLogprobsGrad(torch.autograd.Function):
    """The gradient from inputs that require grad: no constant, so a derivative of it is refused."""
    @staticmethod
    def forward(ctx, *args):
        return _backward(*args)

    @staticmethod
    def backward(ctx, _):
        raise NotImplementedError("token_logprobs_backward has no backward pass: call it under torch.no_grad() or on "
                                  "detached tensors")


def _backward(logits, targets, stats, grad_logprob, grad_entropy, ignore_index):
    z, t, N, V, lead = _rows(logits, targets)
    gl = _row_values(grad_logprob, lead, logits, "grad_logprob")
    gh = None if grad_entropy is None else _row_values(grad_entropy, lead, logits, "grad_entropy")
    stats = _row_values(stats, (*lead, 3), logits, "stats (token_logprobs')")
    return K.token_logprobs_grad(z, t, N, V, int(ignore_index), stats, gl, gh, lead)


def token_logprobs_backward(logits: torch.Tensor, targets: torch.Tensor, stats: torch.Tensor, grad_logprob: torch.Tensor,
                            grad_entropy: Optional[torch.Tensor] = None, ignore_index: int = -100) -> torch.Tensor:
    """The gradient of ``logits`` from the gradients of ``logprob`` and (optionally) ``entropy``, in the
    logits' dtype; ``stats`` is what ``token_logprobs`` returned for the same logits.  It cannot be
    differentiated further."""
    nat.refuse_tangents("token_logprobs_backward", logits, stats, grad_logprob, grad_entropy)
    if torch.is_grad_enabled():
        for t in (logits, stats, grad_logprob, grad_entropy):
            if getattr(t, "requires_grad", False):
                return _TokenLogprobsGrad.apply(logits, targets, stats, grad_logprob, grad_entropy, ignore_index)
    return _backward(logits, targets, stats, grad_logprob, grad_entropy, ignore_index)
