"""The example that runs the packed operators together."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_score_packed_example(dtype):
    path = Path(__file__).resolve().parent.parent / "examples" / "score_packed.py"
    spec = importlib.util.spec_from_file_location("score_packed", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    r = module.run(tokens=9, width=128, inner=160, experts=4, vocab=301, dtype=dtype)
    # h, the logits and the dequantized weights are rounded to dtype: a few units in the last place of values
    # up to 8, summed over 128 columns with random signs
    unit = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    assert r["logprob_error"] < 16 * unit
    assert r["single_error"] < 16 * unit
    assert r["gradient_error"] < 8 * unit
    assert abs(r["perplexity"] / r["plain_perplexity"] - 1) < 16 * unit
