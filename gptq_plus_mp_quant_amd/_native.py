"""ctypes binding of the C ABI in ``include/gptqplus_hip.h`` (library ``_lib/libgptqplus_hip.so``).

The library is the only compute path: if it is missing or cannot be loaded every call raises
``RuntimeError`` -- there is no silent fallback.  ``GPTQPLUS_HIP_LIB`` (environment) names
another build of the same library to load instead (e.g. a variant built for an A/B timing).
"""
from __future__ import annotations

import ctypes
import functools
import os
import re
import struct
from pathlib import Path

import torch
from torch.autograd import forward_ad

LIB_PATH = Path(os.environ.get("GPTQPLUS_HIP_LIB") or
                Path(__file__).resolve().parent / "_lib" / "libgptqplus_hip.so").resolve()
HEADER = Path(__file__).resolve().parent.parent / "include" / "gptqplus_hip.h"

RQ_OK, RQ_EINVAL, RQ_EHIP, RQ_ENOTSUP = 0, -1, -2, -3
RQ_F16, RQ_BF16, RQ_F32 = 0, 1, 2
RQ_QMODE_CHANNEL, RQ_QMODE_STATIC, RQ_QMODE_DYNAMIC = 0, 1, 2
RQ_GMODE_FROZEN, RQ_GMODE_SURROGATE_BLOCK, RQ_GMODE_SURROGATE_ONLINE, RQ_GMODE_BLOCK_GD = 0, 1, 2, 3
RQ_HMATH_SPLIT16, RQ_HMATH_FP32, RQ_HMATH_SPLIT16X3 = 0, 1, 2
RQ_NOALLOC_SCRATCH_BYTES = 128 << 20
RQ_CHOL_MAXBATCH = 64          # matrices per rq_chol_hinv_attempt call
RQ_ACT_ORDER_MAXC = 65536      # widest rq_act_order_perm
RQ_PACKED_MAXBITS = 9          # widest fields the products with packed weights take
RQ_MOE_MAX_EXPERTS, RQ_MOE_MAX_TOP = 1024, 64
RQ_SCORE_MAX_TOP = 64          # alternatives of rq_token_logprobs
RQ_MAX_TOKENS = 1 << 19        # of one call of the products with adapters and of the gated block
RQ_LORA_MAX_RANK, RQ_LORA_MAX_ADAPTERS = 256, 65535
RQ_DISTILL_MAX_TOP = 256       # tokens of a teacher's list
RQ_DISTILL_STATS = 8
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}
TAILS = {"renormalise": 0, "bucket": 1}
# g_update_mode -> (kernel mode of the in-block loop, kernel mode of the trailing update);
# gptq_plus_utils.py:1190 (inner) and :1500 (outer)
GMODES = {"frozen": (RQ_GMODE_FROZEN, RQ_GMODE_FROZEN),
          "surrogate_block": (RQ_GMODE_SURROGATE_BLOCK, RQ_GMODE_SURROGATE_BLOCK),
          "surrogate_online": (RQ_GMODE_SURROGATE_ONLINE, RQ_GMODE_SURROGATE_BLOCK),
          "block_gd": (RQ_GMODE_BLOCK_GD, RQ_GMODE_BLOCK_GD),
          "block_backward": (RQ_GMODE_SURROGATE_ONLINE, RQ_GMODE_FROZEN)}

_P, _I, _L, _D, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_double, ctypes.c_float


class PackedExperts(ctypes.Structure):
    """``rq_packed_experts``: one linear of every expert of a layer."""
    _fields_ = [("qweight", _P), ("scales", _P), ("g_idx", _P), ("ldp", _L), ("lds", _L), ("stride_q", _L),
                ("stride_scales", _L), ("nbits", _I), ("ngroups", _I), ("groupsize", _I)]


# rq_packed_weight, one packed weight, as bytes (made faster than a Structure): qweight, scales, g_idx, ldp, lds, nbits,
# ngroups, groupsize
PACKED_WEIGHT = struct.Struct("PPPqqiii4x")


# name -> (restype, argtypes); mirrors include/gptqplus_hip.h
SIGNATURES = {
    "rq_version": (_I, []),
    "rq_hessian_accum": (_I, [_P, _I, _L, _L, _I, _P, _L, _I, _P, _P, _P, _L, _P]),
    "rq_hessian_accum_noalloc": (_I, [_P, _I, _L, _L, _I, _P, _L, _I, _P, _P, _P]),
    "rq_hessian_workspace_bytes": (_L, [_L, _I, _I, _I]),
    "rq_hessian_math": (_I, [_I]),
    "rq_hessian_timing_events": (_I, [_P, _P]),
    "rq_hessian_accum_multi": (_I, [_P, _I, _L, _L, _I, _I, _P, _P, _P, _P, _P, _L, _P]),
    "rq_hessian_finalize": (_I, [_P, _P, _I, _I, _D, _D, _D, _I, _P, _P]),
    "rq_find_params": (_I, [_P, _I, _I, _I, _L, _I, _I, _I, _I, _P, _P, _P]),
    "rq_find_params_mse": (_I, [_P, _I, _I, _I, _L, _I, _I, _I, _I, _D, _I, _D, _P, _P, _P]),
    "rq_act_order_perm": (_I, [_P, _I, _P, _P, _P]),
    "rq_prepare_subgroup": (_I, [_P, _I, _L, _P, _L, _P, _I, _I, _P, _P, _L, _P, _L, _P, _P]),
    "rq_chol_workspace_bytes": (_L, [_I]),
    "rq_chol_hinv_attempt": (_I, [_P, _I, _I, _P, _P, _P, _P, _P, _P, _P]),
    "rq_gptqplus_terms": (_I, [_P, _L, _P, _P, _P, _I, _I, _I, _D, _D, _I, _P, _P, _P, _L, _P, _P, _P]),
    "rq_quant_block": (_I, [_P, _L, _P, _I, _P, _P, _L, _I, _I, _I, _I, _I, _P, _P, _P, _I, _I,
                            _I, _P, _P, _P, _I, _P, _L, _P, _D, _P]),
    "rq_quant_block_lookahead": (_I, [_P, _L, _P, _I, _I, _I, _I, _I, _P, _I, _I, _P, _P, _P, _I, _I, _I, _P,
                                      _P, _P]),
    "rq_block_loop": (_I, [_P, _L, _P, _I, _I, _I, _I, _I, _P, _P, _P, _I, _I, _I, _P, _P, _L, _P]),
    "rq_trailing_update": (_I, [_P, _L, _P, _P, _L, _P, _I, _I, _I, _I, _I, _P, _P, _I, _I, _P, _L,
                                _P, _D, _P]),
    "rq_writeback": (_I, [_P, _I, _I, _P, _I, _P, _P, _P, _I, _P, _I, _L, _P, _P, _P, _P]),
    "rq_packed_words_per_row": (_L, [_I, _I]),
    "rq_pack_codes": (_I, [_P, _I, _I, _L, _P, _I, _P, _L, _P, _P]),
    "rq_unpack_dequant": (_I, [_P, _I, _I, _L, _I, _P, _L, _P, _P, _I, _L, _P, _P]),
    "rq_current_weight": (_I, [_P, _L, _P, _I, _I, _I, _I, _P, _P, _P, _I, _P, _P, _L, _P, _L, _P]),
    "rq_gather_cols": (_I, [_P, _L, _P, _I, _I, _P, _L, _P]),
    "rq_kfac_curvature": (_I, [_P, _I, _I, _D, _P, _P]),
    "rq_hessian_reg_gemm": (_I, [_P, _L, _P, _I, _I, _I, _I, _P, _L, _P]),
    "rq_block_gd_step": (_I, [_P, _L, _I, _I, _I, _I, _P, _L, _P, _I, _I, _D, _D, _P, _P, _P, _I, _D,
                              _P, _L, _P, _L, _I, _P, _P, _P, _I, _I, _D, _D, _D, _P, _P]),
    "rq_packed_linear": (_I, [_P, _I, _I, _L, _I, _P, _L, _I, _I, _P, _L, _I, _P, _I, _P, _P, _L, _P]),
    "rq_packed_linear_grad_workspace_bytes": (_L, [_I, _I, _I]),
    "rq_packed_linear_grad": (_I, [_P, _I, _I, _L, _I, _P, _L, _I, _I, _P, _L, _I, _P, _I, _P, _L, _P, _L, _P]),
    "rq_packed_moe_workspace_bytes": (_L, [_I, _I, _I, _I, _I]),
    "rq_packed_moe": (_I, [_P, _I, _I, _L, _I, _P, _L, _I, _I, _I, _I, _P, _P, _P, _P, _L, _P, _P, _P, _L, _P]),
    "rq_packed_linear_lora_workspace_bytes": (_L, [_I, _I, _I, _I, _I]),
    "rq_packed_linear_lora": (_I, [_P, _I, _I, _L, _I, _P, _L, _I, _I, _P, _L, _I, _P, _I, _P, _P, _P, _I, _I, _P, _P, _F, _P, _L,
                                   _P, _L, _P]),
    "rq_packed_linear_lora_grad_workspace_bytes": (_L, [_I, _I, _I, _I]),
    "rq_packed_linear_lora_grad": (_I, [_P, _I, _I, _L, _P, _L, _I, _P, _L, _I, _I, _P, _L, _I, _P, _I, _P, _P, _I, _I, _P, _P, _F,
                                        _P, _L, _P, _P, _P, _L, _P]),
    "rq_packed_gated_workspace_bytes": (_L, [_I, _I, _I, _I, _P, _P]),
    "rq_packed_gated": (_I, [_P, _I, _I, _L, _I, _I, _P, _P, _I, _P, _P, _L, _P, _L, _P]),
    "rq_packed_gated_grad_workspace_bytes": (_L, [_I, _I, _I]),
    "rq_packed_gated_grad": (_I, [_P, _I, _I, _L, _I, _P, _I, _P, _P, _I, _P, _L, _P, _L, _P]),
    "rq_distill_loss_workspace_bytes": (_L, [_L, _I]),
    "rq_distill_loss": (_I, [_P, _I, _L, _L, _I, _P, _P, _I, _D, _I, _P, _P, _P, _L, _P]),
    "rq_distill_loss_grad": (_I, [_P, _I, _L, _L, _I, _P, _P, _I, _D, _I, _P, _P, _P, _L, _P]),
    "rq_token_logprobs_workspace_bytes": (_L, [_L, _I, _I]),
    "rq_token_logprobs": (_I, [_P, _I, _L, _L, _I, _P, _L, _I, _P, _P, _P, _P, _P, _P, _L, _P]),
    "rq_token_logprobs_grad": (_I, [_P, _I, _L, _L, _I, _P, _L, _P, _P, _P, _P, _L, _P]),
}

_lib = None


def header_symbols():
    """Function names declared in include/gptqplus_hip.h."""
    text = HEADER.read_text()
    return sorted(set(re.findall(r"^\s*(?:int|int64_t)\s+(rq_\w+)\s*\(", text, re.M)))


def load():
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise RuntimeError(
            f"gptq_plus_mp_quant_amd: HIP library not built ({LIB_PATH}); run "
            "`python -m gptq_plus_mp_quant_amd.build` (hipcc, gfx950)")
    lib = ctypes.CDLL(str(LIB_PATH))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


class Stream(ctypes.c_void_p):
    """A ``hipStream_t`` and the index of its device."""
    index = None


def check(name, rc):
    if rc != RQ_OK:
        raise RuntimeError(f"{name} failed with status {rc}")
    return rc


def call(name, *args):
    """An entry point, on the device of the stream that is its last argument (if it takes one): a kernel goes to
    the current device, and a default stream's handle names none."""
    fn = getattr(load(), name)
    index = args[-1].index if args and isinstance(args[-1], Stream) else None
    if index is None or index == _current_device():
        return check(name, fn(*args))
    with torch.cuda.device(index):
        return check(name, fn(*args))


def on_device_of_first(fn):
    """fn(tensor, ...) with the tensor's device current, as ``call`` has it, for functions that call entry points
    themselves."""
    @functools.wraps(fn)
    def run(t, *args):
        index = t.get_device()
        if index == _current_device():
            return fn(t, *args)
        with torch.cuda.device(index):
            return fn(t, *args)
    return run


def ptr(t):
    """Device pointer of a tensor (None -> NULL)."""
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def stream_of(device):
    s = torch.cuda.current_stream(device)
    out = Stream(s.cuda_stream)
    out.index = s.device.index
    return out


try:
    from torch._C import _cuda_getCurrentRawStream as _raw_stream_of, _cuda_getDevice as _current_device
except ImportError:                                  # a torch without the shortcuts
    _current_device = torch.cuda.current_device

    def _raw_stream_of(index):
        return torch.cuda.current_stream(index).cuda_stream


def raw_stream(t):
    """The current stream of a GPU tensor's device as an int, without making a Stream object (the
    calls on single tokens, whose kernels take a few microseconds, are bound by the host)."""
    return _raw_stream_of(t.get_device())


def refuse_tangents(what, *tensors):
    """The kernels carry no forward-mode tangents on: a tensor with one is refused, not stripped of it."""
    if getattr(forward_ad, "_current_level", 0) < 0:     # no level is open (spares the calls on one token the rest)
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no forward-mode derivative: call it on tensors without tangents")


def save_for_backward(ctx, *tensors):
    """Tensors (or None) that a backward pass takes by saved_for_backward.  Autograd refuses to save those made in inference
    mode; they cannot be changed outside of it and are kept as they are."""
    kept = [t if t is not None and t.is_inference() else None for t in tensors]
    ctx.save_for_backward(*(t if k is None else None for t, k in zip(tensors, kept)))
    ctx.kept = kept


def saved_for_backward(ctx):
    return [t if k is None else k for t, k in zip(ctx.saved_tensors, ctx.kept)]


DTYPE_CODES = {torch.float16: RQ_F16, torch.bfloat16: RQ_BF16, torch.float32: RQ_F32}


def dtype_code(dt):
    if dt == torch.float16:
        return RQ_F16
    if dt == torch.bfloat16:
        return RQ_BF16
    if dt == torch.float32:
        return RQ_F32
    raise TypeError(f"unsupported dtype {dt}; expected float16, bfloat16 or float32")


def require_gpu(t, what):
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise RuntimeError(f"{what} must be a tensor on a ROCm GPU (got "
                           f"{t.device if isinstance(t, torch.Tensor) else type(t)})")
