"""Low-rank adapters beside packed linears: training one, or serving those of many requests over one packed weight.

* ``packed_linear_lora(x, entry, lora_a, lora_b, adapter_ids)`` -- ``W x + b + s B (A x)``, every token with its own
  adapter; differentiable in ``x``, ``lora_a`` and ``lora_b``.
* ``packed_linear_lora_backward(grad_y, x, entry, ...)`` -- the three gradients.

W is the packed weight as ``packed_linear`` reads it.  ``A x`` stays in fp32; the result is rounded once.
"""
from __future__ import annotations

from typing import Dict, Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from . import kernels as K
from .packed import checked_bias, checked_entry, checked_tokens


def _lora(lora_a, lora_b, ids, scaling, x, R, C, lead):
    """(lora_a, lora_b, n, r, ids or None, scaling tensor or None, scale), each tensor contiguous."""
    dev, dt = x.get_device(), x.dtype
    for t, name in ((lora_a, "lora_a"), (lora_b, "lora_b")):
        if not isinstance(t, torch.Tensor) or t.dtype is not dt or t.get_device() != dev:
            raise ValueError(f"{name} must be a {dt} tensor on {x.device}")
    sa, sb = lora_a.shape, lora_b.shape
    if len(sa) not in (2, 3) or len(sb) != len(sa) or sa[-1] != C or sb[-2] != R or sa[-2] != sb[-1] or sa[0] != (sb[0] if len(sa) == 3 else sa[0]):
        raise ValueError(f"lora_a and lora_b must be [n, r, {C}] and [n, {R}, r] (or [r, {C}] and [{R}, r]), got {tuple(sa)} and {tuple(sb)}")
    n, r = sa[0] if len(sa) == 3 else 1, sa[-2]
    if not 1 <= n <= nat.RQ_LORA_MAX_ADAPTERS or not 1 <= r <= nat.RQ_LORA_MAX_RANK:
        raise ValueError(f"{n} adapters of rank {r}: 1 to {nat.RQ_LORA_MAX_ADAPTERS} of rank 1 to {nat.RQ_LORA_MAX_RANK} are supported")
    if ids is None:
        if n != 1:
            raise ValueError(f"adapter_ids are needed to choose between {n} adapters")
    elif not isinstance(ids, torch.Tensor) or ids.dtype is not torch.int64 or ids.shape != lead or ids.get_device() != dev:
        raise ValueError(f"adapter_ids must be int64 {list(lead)} on {x.device}")
    elif not ids.is_contiguous():
        ids = ids.contiguous()
    scale = 1.0
    if isinstance(scaling, torch.Tensor):
        if scaling.dtype is not torch.float32 or scaling.shape != (n,) or scaling.get_device() != dev:
            raise ValueError(f"scaling must be a number or float32 [{n}] on {x.device}")
        if scaling.requires_grad and torch.is_grad_enabled():
            raise ValueError("scaling is constant and would get no gradient; detach it")
        scaling = scaling.contiguous()
    else:
        scaling, scale = None, float(scaling)
    return lora_a.contiguous(), lora_b.contiguous(), n, r, ids, scaling, scale


def _needs_grad(*tensors):
    for t in tensors:                                # a loop: any() over a generator takes three times as long
        if getattr(t, "requires_grad", False):
            return True
    return False


def _tokens_ok(T):
    if T > nat.RQ_MAX_TOKENS:
        raise ValueError(f"{T} tokens: at most {nat.RQ_MAX_TOKENS} in one call")


def _forward(x, entry, lora_a, lora_b, ids, scaling, bias):
    q, nbits, scales, R, C, ng, g_idx, groupsize = checked_entry(entry, 0)
    x2, T, lead = checked_tokens(x, C, q, "x")
    _tokens_ok(T)
    adapters = _lora(lora_a, lora_b, ids, scaling, x, R, C, lead)
    return K.packed_linear_lora(x2, q, nbits, scales, T, R, C, ng, g_idx, groupsize, checked_bias(bias, x, R), *adapters, lead)


def _backward(grad_y, x, entry, lora_a, lora_b, ids, scaling, want_x=True, want_lora=True):
    q, nbits, scales, R, C, ng, g_idx, groupsize = checked_entry(entry, 0)
    g2, T, lead = checked_tokens(grad_y, R, q, "grad_y")
    x2, _, lead_x = checked_tokens(x, C, q, "x")
    if lead != lead_x or x.dtype != grad_y.dtype:
        raise ValueError(f"x must be {grad_y.dtype} {[*lead, C]}, got {x.dtype} {list(x.shape)}")
    _tokens_ok(T)
    a, b, *rest = _lora(lora_a, lora_b, ids, scaling, x, R, C, lead)
    return K.packed_linear_lora_grad(g2, x2, q, nbits, scales, T, R, C, ng, g_idx, groupsize, a, b, *rest, lead, want_x, want_lora)


class _PackedLinearLora(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, lora_a, lora_b, entry, ids, scaling, bias):
        y = _forward(x, entry, lora_a, lora_b, ids, scaling, bias)
        # the tensors, not the dict, as packed_linear saves them
        nat.save_for_backward(ctx, x, lora_a, lora_b, entry["qweight"], entry["scales"], entry["g_idx"], ids,
                              scaling if isinstance(scaling, torch.Tensor) else None)
        ctx.scaling = scaling if not isinstance(scaling, torch.Tensor) else None
        ctx.fields = dict(nbits=entry["nbits"], groupsize=entry.get("groupsize", 0))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        x, lora_a, lora_b, q, scales, g_idx, ids, scaling = nat.saved_for_backward(ctx)
        need = ctx.needs_input_grad
        gx, ga, gb = _backward(grad_y, x, dict(qweight=q, scales=scales, g_idx=g_idx, **ctx.fields), lora_a, lora_b, ids,
                               ctx.scaling if scaling is None else scaling, need[0], need[1] or need[2])
        return gx, ga if need[1] else None, gb if need[2] else None, None, None, None, None


def packed_linear_lora(x: torch.Tensor, entry: Dict[str, object], lora_a: torch.Tensor, lora_b: torch.Tensor,
                       adapter_ids: Optional[torch.Tensor] = None, scaling: Union[float, torch.Tensor] = 1.0,
                       bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``packed_linear(x, entry, bias)`` with a low-rank adapter for every token: ``x [..., C]`` -> ``[..., R]``,
    ``W x + bias + s B (A x)``, in x's dtype (fp16, bf16 or fp32).

    ``lora_a`` [n, r, C] and ``lora_b`` [n, R, r] (x's dtype; r up to 256, n up to 65535) hold n adapters, ``adapter_ids`` [...] (int64) says
    which is whose: a token with an id below 0 has none, one with an id from n on gets NaN.  Without ids there is one
    adapter (which may come as [r, C] and [R, r]) for all tokens.  ``scaling``: a number, or fp32 [n].

    Differentiable in ``x``, ``lora_a`` and ``lora_b``; the packed weight, the bias and the scaling are constants
    (ones that require grad are refused), forward-mode tangents are refused.  Made for few tokens, as
    ``packed_linear`` is; at most 2^19."""
    nat.refuse_tangents("packed_linear_lora", x, lora_a, lora_b, scaling, bias, entry["scales"])
    if torch.is_grad_enabled():
        if bias is not None and getattr(bias, "requires_grad", False):
            raise ValueError("packed_linear_lora: the bias of a packed linear is a constant; detach it")
        if isinstance(scaling, torch.Tensor) and scaling.requires_grad:
            raise ValueError("scaling is constant and would get no gradient; detach it")
        if _needs_grad(x, lora_a, lora_b):
            checked_entry(entry, 0)                  # under autograd; forward runs without
            return _PackedLinearLora.apply(x, lora_a, lora_b, entry, adapter_ids, scaling, bias)
    return _forward(x, entry, lora_a, lora_b, adapter_ids, scaling, bias)


class _PackedLinearLoraGrad(torch.autograd.Function):
    """The gradients from inputs that require grad: no constants, so a derivative of them is refused."""
    @staticmethod
    def forward(ctx, grad_y, x, lora_a, lora_b, entry, ids, scaling):
        return _backward(grad_y, x, entry, lora_a, lora_b, ids, scaling)

    @staticmethod
    def backward(ctx, *_):
        raise NotImplementedError("packed_linear_lora_backward has no backward pass: call it under torch.no_grad() or on "
                                  "detached tensors")


def packed_linear_lora_backward(grad_y: torch.Tensor, x: torch.Tensor, entry: Dict[str, object], lora_a: torch.Tensor,
                                lora_b: torch.Tensor, adapter_ids: Optional[torch.Tensor] = None,
                                scaling: Union[float, torch.Tensor] = 1.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients of ``packed_linear_lora``'s x, lora_a and lora_b from the gradient of its result, in their shapes and
    dtype; an adapter that no token has gets 0.  The results do not change from run to run.  They cannot be
    differentiated further."""
    nat.refuse_tangents("packed_linear_lora_backward", grad_y, x, lora_a, lora_b, scaling, entry["scales"])
    if torch.is_grad_enabled() and _needs_grad(grad_y, x, lora_a, lora_b):
        checked_entry(entry, 0)
        return _PackedLinearLoraGrad.apply(grad_y, x, lora_a, lora_b, entry, adapter_ids, scaling)
    return _backward(grad_y, x, entry, lora_a, lora_b, adapter_ids, scaling)
