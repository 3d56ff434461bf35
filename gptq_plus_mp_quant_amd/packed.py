"""Running a quantised model from its packed entries.

``export_packed`` leaves a linear as codes, scales and the scale group of every column.  The functions
here compute with that form; the dequantized weight is never written out:

* ``packed_linear(x, entry)`` -- ``x W^T`` (+ bias) for a few tokens; differentiable in ``x``.
* ``packed_linear_backward(grad_y, entry)`` -- the gradient of ``x`` alone.
* ``packed_gated(x, gate, up)`` -- the gated half of a feed-forward block, ``act(gate(x)) * up(x)``; differentiable in
  ``x``.
* ``packed_gated_backward(grad_h, pre, gate, up)`` -- the gradient of its ``x`` alone.
* ``packed_moe(x, router, gate, up, down, top_k)`` -- a mixture-of-experts layer whose experts' linears
  are packed, each of the three stacked over the experts by ``stack_packed``.

W is scale times code as the entry holds them (``dequantize_packed`` rounds that product to the
layer's type; the products here do not).  Sums are fp32 and the result is rounded once, to x's type.
An entry's ``groupsize`` (``export_packed`` adds it where the groups are runs of columns) says that
column c is in group ``c // groupsize``; without it every column's group is read from ``g_idx``.
"""
from __future__ import annotations

from typing import Dict, Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from . import kernels as K


def _rows_apart(t):
    """A single row whose stride, which no element needs, is shorter than the row."""
    return t.clone(memory_format=torch.contiguous_format)


def checked_entry(entry: Dict[str, object], batch: int):
    """(qweight, nbits, scales, R, C, ngroups, g_idx, groupsize) of an entry (batch = 1: stacked over
    experts)."""
    q, scales, g_idx, nbits = entry["qweight"], entry["scales"], entry["g_idx"], entry["nbits"]
    groupsize = entry.get("groupsize", 0)
    dev = q.get_device()
    if dev < 0 or scales.get_device() != dev or g_idx.get_device() != dev:
        for t, name in ((q, "qweight"), (scales, "scales"), (g_idx, "g_idx")):
            nat.require_gpu(t, f"packed entry: {name}")
        raise ValueError("packed entry: qweight, scales and g_idx are on different devices")
    if scales.requires_grad and torch.is_grad_enabled():
        raise ValueError("packed entry: the scales are constants and would get no gradient; detach them")
    if q.dtype is not torch.int32 or scales.dtype is not torch.float32 or g_idx.dtype is not torch.int32:
        raise ValueError("packed entry: qweight and g_idx must be int32, scales float32")
    if not 2 <= nbits <= nat.RQ_PACKED_MAXBITS:
        raise NotImplementedError(f"packed weights of {nbits} bits: 2 to {nat.RQ_PACKED_MAXBITS} are supported")
    qs, ss, gs = q.shape, scales.shape, g_idx.shape
    if len(qs) != 2 + batch or len(ss) != 2 + batch or len(gs) != 1 + batch:
        raise ValueError("packed entry: qweight [R, words], scales [ngroups, R] and g_idx [C] are expected"
                         + (", each with a leading expert dimension (stack_packed)" if batch else ""))
    R, words, ng, C = qs[-2], qs[-1], ss[-2], gs[-1]
    if C == 0 or R == 0 or ng == 0 or words * 32 < C * nbits or ss[-1] != R:
        raise ValueError("packed entry: the shapes of qweight, scales and g_idx do not belong together")
    if batch and not qs[0] == ss[0] == gs[0]:
        raise ValueError("packed entry: qweight, scales and g_idx hold different numbers of experts")
    if groupsize < 0 or (groupsize and ng > 1 and (C - 1) // groupsize >= ng):
        raise ValueError(f"packed entry: groupsize {groupsize} does not fit {ng} groups of {C} columns")
    qst, sst = q.stride(), scales.stride()
    # strides along a dimension of one element are never used, whatever they are
    if (qst[-1] != 1 and words > 1) or (sst[-1] != 1 and R > 1) or (qst[-2] < words and R > 1) or (sst[-2] < R and ng > 1):
        raise ValueError("packed entry: qweight and scales need unit column strides")
    return (q if qst[-2] >= words else _rows_apart(q), nbits, scales if sst[-2] >= R else _rows_apart(scales), R, C, ng,
            g_idx if g_idx.is_contiguous() else g_idx.contiguous(), groupsize)


def checked_tokens(x, width, q, name):
    """x as [T, width] with unit column stride (copied only if its strides need it), T, and x's leading
    dimensions."""
    if not (isinstance(x, torch.Tensor) and x.is_cuda):
        nat.require_gpu(x, name)
    if x.dtype not in nat.DTYPE_CODES:
        raise TypeError(f"{name}: unsupported dtype {x.dtype}; expected float16, bfloat16 or float32")
    shape = x.shape
    if len(shape) < 1 or shape[-1] != width:
        raise ValueError(f"{name} must be [..., {width}], got {tuple(shape)}")
    if x.get_device() != q.get_device():
        raise ValueError(f"{name} is on {x.device}, the packed weight on {q.device}")
    x2 = x if len(shape) == 2 else x.reshape(-1, width)
    T = x2.shape[0]
    s0, s1 = x2.stride()
    if s1 != 1 or s0 < width:
        if T > 1 or s1 != 1:
            x2 = x2.contiguous()
        if x2.stride(0) < width:                 # one token: its row stride is never used
            x2 = x2.as_strided((T, width), (width, 1))
    return x2, T, (T,) if x2 is x else shape[:-1]


def checked_bias(bias, x, R):
    if bias is None:
        return None
    if not isinstance(bias, torch.Tensor) or bias.dtype != x.dtype or bias.shape != (R,) or bias.device != x.device:
        raise ValueError(f"bias must be {x.dtype} [{R}] on {x.device}")
    return bias.contiguous()


class _PackedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, entry, bias):
        y = _forward(x, entry, bias)
        # the tensors, not the dict: the gradient goes through the weight of this call.  Tensors made in inference
        # mode cannot be saved (nor changed outside of it).
        weight = entry["qweight"], entry["scales"], entry["g_idx"]
        ctx.unsaved = weight if any(t.is_inference() for t in weight) else None
        ctx.save_for_backward(*(() if ctx.unsaved else weight))
        ctx.fields = dict(nbits=entry["nbits"], groupsize=entry.get("groupsize", 0))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        q, scales, g_idx = ctx.unsaved or ctx.saved_tensors
        return _backward(grad_y, dict(qweight=q, scales=scales, g_idx=g_idx, **ctx.fields)), None, None


def _forward(x, entry, bias):
    q, nbits, scales, R, C, ng, g_idx, groupsize = checked_entry(entry, 0)
    x2, T, lead = checked_tokens(x, C, q, "x")
    return K.packed_linear(x2, q, nbits, scales, T, R, C, ng, g_idx, groupsize, checked_bias(bias, x, R), lead)


def packed_linear(x: torch.Tensor, entry: Dict[str, object], bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x [..., C]`` times the transpose of a packed weight, ``[..., R]`` in x's dtype (fp16, bf16 or
    fp32); ``bias`` [R] of the same dtype is added before the rounding.  Any number of tokens; the
    kernels are made for few (a decoding step, a short prompt).  Differentiable in ``x``; the weight
    and the bias are constants (scales or a bias that require grad are refused).  Forward-mode tangents are
    refused."""
    nat.refuse_tangents("packed_linear", x, bias, entry["scales"])
    if torch.is_grad_enabled():
        if bias is not None and getattr(bias, "requires_grad", False):
            raise ValueError("packed_linear: the bias of a packed linear is a constant; detach it")
        if isinstance(x, torch.Tensor) and x.requires_grad:
            checked_entry(entry, 0)                       # under autograd; forward runs without
            return _PackedLinear.apply(x, entry, bias)
    return _forward(x, entry, bias)


class _PackedLinearGrad(torch.autograd.Function):
    """The gradient of a grad_y that requires grad: no constant, so a derivative of it is refused."""
    @staticmethod
    def forward(ctx, grad_y, entry):
        return _backward(grad_y, entry)

    @staticmethod
    def backward(ctx, _):
        raise NotImplementedError("packed_linear_backward has no backward pass: call it under torch.no_grad() or on "
                                  "detached tensors")


def _backward(grad_y, entry):
    q, nbits, scales, R, C, ng, g_idx, groupsize = checked_entry(entry, 0)
    g2, T, lead = checked_tokens(grad_y, R, q, "grad_y")
    return K.packed_linear_grad(g2, q, nbits, scales, T, R, C, ng, g_idx, groupsize, lead)


def packed_linear_backward(grad_y: torch.Tensor, entry: Dict[str, object]) -> torch.Tensor:
    """The gradient of ``packed_linear``'s x: ``grad_y [..., R]`` times the packed weight, ``[..., C]`` in
    grad_y's dtype.  The result does not change from run to run.  It cannot be differentiated further."""
    nat.refuse_tangents("packed_linear_backward", grad_y, entry["scales"])
    if torch.is_grad_enabled() and isinstance(grad_y, torch.Tensor) and grad_y.requires_grad:
        checked_entry(entry, 0)
        return _PackedLinearGrad.apply(grad_y, entry)
    return _backward(grad_y, entry)


def _pair(gate, up, name):
    """The checked tensors of gate and up, I and C."""
    g, u = checked_entry(gate, 0), checked_entry(up, 0)
    if g[3] != u[3] or g[4] != u[4]:
        raise ValueError(f"{name}: gate and up must have one shape, got {g[3]} x {g[4]} and {u[3]} x {u[4]}")
    if g[0].get_device() != u[0].get_device():
        raise ValueError(f"{name}: gate and up are on different devices")
    return (*g[:3], *g[5:]), (*u[:3], *u[5:]), g[3], g[4]


def _activation(activation):
    if activation not in nat.ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(nat.ACTIVATIONS)}, got {activation!r}")
    return nat.ACTIVATIONS[activation]


def _gated(x, gate, up, activation, want_pre):
    g, u, I, C = _pair(gate, up, "packed_gated")
    x2, T, lead = checked_tokens(x, C, g[0], "x")
    if T > nat.RQ_MAX_TOKENS:
        raise ValueError(f"packed_gated: {T} tokens, at most {nat.RQ_MAX_TOKENS} in one call")
    return K.packed_gated(x2, g, u, T, I, C, _activation(activation), want_pre, lead)


def _gated_backward(grad_h, pre, gate, up, activation):
    g, u, I, C = _pair(gate, up, "packed_gated_backward")
    g2, T, lead = checked_tokens(grad_h, I, g[0], "grad_h")
    if T > nat.RQ_MAX_TOKENS:
        raise ValueError(f"packed_gated_backward: {T} tokens, at most {nat.RQ_MAX_TOKENS} in one call")
    if not isinstance(pre, torch.Tensor) or pre.dtype is not torch.float32 or pre.shape != (*lead, 2, I) or \
            pre.get_device() != grad_h.get_device():
        raise ValueError(f"pre (packed_gated's) must be float32 {[*lead, 2, I]} on {grad_h.device}")
    return K.packed_gated_grad(g2, pre.contiguous(), g, u, T, I, C, _activation(activation), lead)


class _PackedGated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, up, activation):
        h, pre = _gated(x, gate, up, activation, True)
        # the tensors, not the dicts, as in _PackedLinear
        weights = [e[k] for e in (gate, up) for k in ("qweight", "scales", "g_idx")]
        ctx.unsaved = weights if any(t.is_inference() for t in weights) else None
        ctx.save_for_backward(pre, *(() if ctx.unsaved else weights))
        ctx.fields = [dict(nbits=e["nbits"], groupsize=e.get("groupsize", 0)) for e in (gate, up)]
        ctx.activation = activation
        ctx.mark_non_differentiable(pre)
        ctx.set_materialize_grads(False)                 # or backward gets zeros of pre's size
        return h, pre

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_h, _):
        if grad_h is None:
            return None, None, None, None
        pre, *weights = ctx.saved_tensors
        weights = ctx.unsaved or weights
        gate, up = (dict(zip(("qweight", "scales", "g_idx"), weights[3 * k:]), **f) for k, f in enumerate(ctx.fields))
        return _gated_backward(grad_h, pre, gate, up, ctx.activation), None, None, None


def packed_gated(x: torch.Tensor, gate: Dict[str, object], up: Dict[str, object], activation: str = "silu",
                 return_pre: bool = False):
    """The gated half of a feed-forward block in one pass over its weights: ``x [..., C]`` -> ``act(x Wg^T) * (x Wu^T)``,
    ``[..., I]`` in x's dtype (fp16, bf16 or fp32); ``packed_linear`` with the down projection completes it.

    ``gate`` and ``up`` are entries of one shape, each with bits and groups of its own (one launch where those
    agree).  ``activation``: "silu", "gelu" (erf) or "gelu_tanh".  Sums and products are fp32, rounded once.  ``return_pre``
    adds both projections, fp32 ``[..., 2, I]``, for ``packed_gated_backward``.

    Differentiable in ``x`` (not through ``pre``); the weights are constants, forward-mode tangents are refused.  Made for few
    tokens, as ``packed_linear`` is; at most 2^19."""
    nat.refuse_tangents("packed_gated", x, gate["scales"], up["scales"])
    if torch.is_grad_enabled() and isinstance(x, torch.Tensor) and x.requires_grad:
        _pair(gate, up, "packed_gated")              # under autograd; forward runs without
        h, pre = _PackedGated.apply(x, gate, up, activation)
    else:
        h, pre = _gated(x, gate, up, activation, return_pre)
    return (h, pre) if return_pre else h


class _PackedGatedGrad(torch.autograd.Function):
    """The gradient from inputs that require grad: no constant, so a derivative of it is refused."""
    @staticmethod
    def forward(ctx, grad_h, pre, gate, up, activation):
        return _gated_backward(grad_h, pre, gate, up, activation)

    @staticmethod
    def backward(ctx, _):
        raise NotImplementedError("packed_gated_backward has no backward pass: call it under torch.no_grad() or on "
                                  "detached tensors")


def packed_gated_backward(grad_h: torch.Tensor, pre: torch.Tensor, gate: Dict[str, object], up: Dict[str, object],
                          activation: str = "silu") -> torch.Tensor:
    """The gradient of ``packed_gated``'s x from the gradient of its result ``[..., I]``, in grad_h's dtype; ``pre`` is what
    ``packed_gated(..., return_pre=True)`` returned beside it.  The result does not change from run to run.  It cannot be
    differentiated further."""
    nat.refuse_tangents("packed_gated_backward", grad_h, pre, gate["scales"], up["scales"])
    if torch.is_grad_enabled() and (getattr(grad_h, "requires_grad", False) or getattr(pre, "requires_grad", False)):
        _pair(gate, up, "packed_gated_backward")
        return _PackedGatedGrad.apply(grad_h, pre, gate, up, activation)
    return _gated_backward(grad_h, pre, gate, up, activation)


def stack_packed(entries: Sequence[Dict[str, object]]) -> Dict[str, object]:
    """One linear of every expert as one entry, for ``packed_moe``: qweight [E, R, words], scales
    [E, ngroups, R], g_idx [E, C].  The experts' entries must agree in shape, bits and number of
    groups."""
    entries = list(entries)
    if not entries:
        raise ValueError("stack_packed: no entries")
    first = entries[0]
    for e in entries:
        checked_entry(e, 0)
        if int(e["nbits"]) != int(first["nbits"]) or e["qweight"].shape != first["qweight"].shape or \
                e["scales"].shape != first["scales"].shape or e["g_idx"].shape != first["g_idx"].shape:
            raise ValueError("stack_packed: the experts' entries differ in bits, shape or groups")
    out = {k: torch.stack([e[k] for e in entries]) for k in ("qweight", "scales", "g_idx")}
    sizes = {int(e.get("groupsize", 0)) for e in entries}
    out.update(nbits=int(first["nbits"]), bits=first.get("bits"), sym=first.get("sym"), shape=tuple(first["shape"]),
               dtype=first["dtype"], groupsize=sizes.pop() if len(sizes) == 1 else 0)
    return out


def packed_moe(x: torch.Tensor, router: torch.Tensor, gate: Dict[str, object], up: Dict[str, object],
               down: Dict[str, object], top_k: int, norm_topk: bool = True, return_routing: bool = False):
    """A mixture-of-experts layer for a few tokens: ``x [..., D]`` -> ``[..., D]`` in x's dtype.

    ``router`` [E, D] (x's dtype) gives the logits; each token goes to its ``top_k`` largest (equal
    logits: the lowest index), weighted by the softmax over all experts, divided by the chosen ones' sum
    with ``norm_topk``; an expert is ``down(silu(gate(x)) * up(x))``.  ``gate`` / ``up`` (I x D) and ``down``
    (D x I) are stacked entries, each with bits and groups of its own.  ``return_routing`` adds the
    chosen ids (int32) and weights (fp32), ``[..., top_k]``.  At most 1024 experts, 64 chosen.  It has
    no backward pass: an x that requires grad is refused, and forward-mode tangents are."""
    nat.refuse_tangents("packed_moe", x, router, gate["scales"], up["scales"], down["scales"])
    if torch.is_grad_enabled() and (getattr(x, "requires_grad", False) or getattr(router, "requires_grad", False)):
        raise NotImplementedError("packed_moe has no backward pass: call it under torch.no_grad() or on detached tensors")
    g, u, d = checked_entry(gate, 1), checked_entry(up, 1), checked_entry(down, 1)
    E, I, D = g[0].shape[0], g[3], g[4]
    if u[0].shape[0] != E or d[0].shape[0] != E or u[3] != I or u[4] != D or d[3] != D or d[4] != I:
        raise ValueError("packed_moe: gate and up must be [E, I x D] and down [E, D x I]")
    if not u[0].get_device() == d[0].get_device() == g[0].get_device():
        raise ValueError("packed_moe: gate, up and down are on different devices")
    x2, T, _ = checked_tokens(x, D, g[0], "x")
    if not isinstance(router, torch.Tensor) or router.shape != (E, D) or router.dtype != x.dtype or router.device != x.device:
        raise ValueError(f"packed_moe: router must be {x.dtype} [{E}, {D}] on {x.device}")
    top_k = int(top_k)
    if E > nat.RQ_MOE_MAX_EXPERTS or not 1 <= top_k <= min(E, nat.RQ_MOE_MAX_TOP):
        raise ValueError(f"packed_moe: top_k {top_k} of {E} experts (at most {nat.RQ_MOE_MAX_TOP} of "
                         f"{nat.RQ_MOE_MAX_EXPERTS})")
    r0, r1 = router.stride()
    if r1 != 1 or r0 < D:
        router = router.contiguous()
        if router.stride(0) < D:
            router = router.as_strided((E, D), (D, 1))
    args = [(q, nbits, scales, ng, gi, gs) for q, nbits, scales, _, _, ng, gi, gs in (g, u, d)]
    y, ids, weights = K.packed_moe(x2, router, T, D, I, E, *args, top_k, norm_topk, return_routing)
    y = y if x.dim() == 2 else y.view(x.shape)
    if not return_routing:
        return y
    lead = x.shape[:-1]
    return y, ids.view(*lead, top_k), weights.view(*lead, top_k)
