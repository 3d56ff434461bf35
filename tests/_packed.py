"""Packed entries for the tests, and the products with them in 64 bits."""
from __future__ import annotations

import numpy as np
import torch

from oracle.packing import pack_rows
from tests._util import rng

# unit roundoff of the output types, and half of fp16's smallest subnormal
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}


def make_entry(seed, R, C, nbits, groups, batch=None):
    """A random entry on the CPU (every code value occurs) and its weight in float64 [R, C].  groups:
    "channel", a group size, or "order<size>" for groups of permuted columns (no "groupsize")."""
    r = rng(seed)
    if batch is not None:
        each = [make_entry(seed + 1000 * (i + 1), R, C, nbits, groups) for i in range(batch)]
        out = dict(each[0][0])
        for k in ("qweight", "scales", "g_idx"):
            out[k] = torch.stack([e[k] for e, _ in each])
        return out, torch.stack([w for _, w in each])
    half = 1 << (nbits - 1)
    codes = r.integers(-half, half, size=(R, C))
    size = C if groups == "channel" else int(str(groups).replace("order", ""))
    ng = -(-C // size)
    order = r.permutation(C) if str(groups).startswith("order") else np.arange(C)
    g_idx = (np.argsort(order) // size).astype(np.int32)
    scales = (r.lognormal(0.0, 0.5, size=(ng, R)) * 0.02).astype(np.float32)
    w = scales.astype(np.float64)[g_idx].T * codes
    entry = dict(qweight=torch.from_numpy(pack_rows(codes, nbits).view(np.int32)), scales=torch.from_numpy(scales),
                 g_idx=torch.from_numpy(g_idx), nbits=nbits, bits=nbits, sym=True, shape=(R, C), dtype="float16")
    if not str(groups).startswith("order"):
        entry["groupsize"] = size
    return entry, torch.from_numpy(w)


def on(entry, dev):
    return {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in entry.items()}


def sum_eps(n):
    """A bound of an fp32 sum's error over the sum of its terms' magnitudes: rounding errors of either
    sign grow like sqrt(n), and 32 covers the few-term sums and the products."""
    return (32.0 + n ** 0.5) * 2.0 ** -24


def assert_within(got, want, bound, what):
    """got (any type) against want (float64), element by element; non-finite values have to match."""
    got = got.detach().cpu().double()
    fin = torch.isfinite(want)
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = ~fin & ~torch.isnan(want)
    assert torch.equal(got[inf], want[inf]), what
    over = ((got - want).abs() - bound)[fin]
    assert over.numel() == 0 or float(over.max()) <= 0.0, f"{what}: {float(over.max())} over the bound"
