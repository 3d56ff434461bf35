"""The example that trains adapters on a packed model and serves them: the operators together, as they are used."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tail", ["bucket", "renormalise"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_adapt_packed_example(dtype, tail):
    path = Path(__file__).resolve().parent.parent / "examples" / "adapt_packed.py"
    spec = importlib.util.spec_from_file_location("adapt_packed", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    r = module.run(tokens=19, width=128, inner=160, vocab=301, rank=5, steps=2, top_k=12, dtype=dtype, tail=tail)
    # each rounding is off by at most half a unit; h, the block's result, the logits' gradient, the dequantized weights and
    # the gradients themselves are rounded to dtype one after the other, and the logits' rounding, of values up to 32, is an
    # error of the probabilities: 2 units for each of six, 16 for the logits.  The gradient is a difference of
    # probabilities, and each of them is off by as much.
    unit = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[dtype]
    if dtype == torch.float32:
        unit = 2.0 ** -18                       # sums of up to 301 terms, 32 + sqrt(301) roundings each
    assert abs(r["loss"] - r["plain_loss"]) <= 28 * unit * max(1.0, r["plain_loss"])
    assert max(r["gradient_errors"]) <= 28 * unit * r["terms"]
    assert r["serving_error"] <= 4 * unit
    assert len(r["losses"]) == 3 and all(math.isfinite(v) for v in r["losses"])
