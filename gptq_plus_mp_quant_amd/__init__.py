"""MI355X (gfx950) implementation of the GPTQ+ per-linear quantization hot path.

``GPTQPlus``, ``GPTQ`` and ``WeightQuantizer`` are drop-ins for the reference classes of the
same names; all arithmetic runs in the HIP library built by ``gptq_plus_mp_quant_amd.build``.
``packed_linear`` / ``packed_gated`` / ``packed_moe`` run a model from its packed entries, ``packed_linear_lora`` with
low-rank adapters beside them; ``token_logprobs`` scores what it answers, and ``distillation_loss`` compares that with a
teacher's best tokens.
"""
from .adapters import packed_linear_lora, packed_linear_lora_backward
from .distillation import Distillation, distillation_loss, distillation_loss_backward
from .export import dequantize_packed, export_packed, load_packed, save_packed
from .gptq import GPTQ
from .gptq_plus import GPTQPlus, add_batch_shared, fasterquant_shared
from .packed import (packed_gated, packed_gated_backward, packed_linear, packed_linear_backward, packed_moe,
                     stack_packed)
from .quant_utils import WeightQuantizer, get_minq_maxq
from .scoring import TokenLogprobs, token_logprobs, token_logprobs_backward

__all__ = ["GPTQPlus", "GPTQ", "WeightQuantizer", "add_batch_shared", "fasterquant_shared", "get_minq_maxq",
           "export_packed",
           "dequantize_packed", "save_packed", "load_packed",
           "packed_linear", "packed_linear_backward", "packed_moe", "stack_packed", "packed_gated", "packed_gated_backward",
           "packed_linear_lora", "packed_linear_lora_backward",
           "Distillation", "distillation_loss", "distillation_loss_backward",
           "TokenLogprobs", "token_logprobs", "token_logprobs_backward"]
__version__ = "0.1.0"
