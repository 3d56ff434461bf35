"""Operators that run and score a quantised model, as cases that can be timed and checked.

``export_packed`` stores a quantised linear as an nbits-wide bitstream of codes per row, a
[ngroups, R] table of scales and the scale group of every column.  The operators here work on that
form, and score what the model answers:

  linear     packed_linear: x W^T for a few tokens, W read as packed codes
  lineargrad packed_linear_backward: the gradient of x through the same weight
  moe        packed_moe: a mixture-of-experts layer (router, top-k, gate / up, SiLU, down) for a few
             tokens, every expert's linears packed
  score      token_logprobs: log probabilities of given tokens, the entropy and the top alternatives
  scoregrad  token_logprobs_backward: the gradient of the logits

A case is a dict of plain values.  "groups" says how the scales of a weight lie: "channel" (one per
row), a group size (consecutive columns), or "order<size>" (groups of the act_order's permuted
columns, so a group's columns are spread over the row).
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # Generation, one token: an attention projection of a 4096-wide model, w4 symmetric with
        # 128-column groups.  Latency is all there is.
        dict(name="linear_token", kind="linear", T=1, R=4096, C=4096, nbits=4, groups="128", dtype="bf16", bias=False),
        # A ragged linear (no size a multiple of anything) from fp32 activations: w4 asymmetric (5
        # stored bits) with groups along the act_order, a handful of tokens, with a bias.
        dict(name="linear_ragged", kind="linear", T=7, R=1026, C=1365, nbits=5, groups="order128", dtype="fp32", bias=True),
        # A 70B model's down projection for a batch of 16 sequences: the largest weight.
        dict(name="linear_batch", kind="linear", T=16, R=8192, C=28672, nbits=4, groups="128", dtype="bf16", bias=False),
        # w4 asymmetric per channel (the quantizer's common form), the end of a short prompt in fp16.
        dict(name="lineargrad_short", kind="lineargrad", T=8, R=4096, C=4096, nbits=5, groups="channel", dtype="fp16", bias=False),
        # The gradient through an 8B model's gate projection, 64 tokens.
        dict(name="lineargrad_wide", kind="lineargrad", T=64, R=14336, C=4096, nbits=4, groups="128", dtype="bf16", bias=False),
        # One token through 128 small experts, 8 of them chosen.
        dict(name="moe_token", kind="moe", T=1, D=2048, I=768, E=128, K=8, nbits=4, groups="128", dtype="bf16", norm=True),
        # A batch of 32 through 8 large experts, 2 chosen: every expert is read, for about 8 tokens.
        dict(name="moe_batch", kind="moe", T=32, D=4096, I=7168, E=8, K=2, nbits=5, groups="channel", dtype="fp16", norm=True),
        # One sampled token over a 128256-entry vocabulary, 20 alternatives.
        dict(name="score_token", kind="score", N=1, V=128256, top=20, dtype="bf16", masked=0.0),
        # Scoring a prompt of 2048 tokens, 5 alternatives each.
        dict(name="score_prompt", kind="score", N=2048, V=128256, top=5, dtype="bf16", masked=0.0),
        # Constrained answers in fp32: most of an odd vocabulary masked, some rows with nothing left.
        dict(name="score_masked", kind="score", N=37, V=32003, top=8, dtype="fp32", masked=0.7),
        # The gradient for a few answers, fp32 logits.
        dict(name="scoregrad_few", kind="scoregrad", N=12, V=32003, top=0, dtype="fp32", masked=0.3),
        # The gradient of a calibration sample's loss: 1024 tokens.
        dict(name="scoregrad_sample", kind="scoregrad", N=1024, V=128256, top=0, dtype="bf16", masked=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width between lo and hi: a multiple of 128 or of 8 as model widths are, or any number."""
    c = _log(rng, lo, hi)
    m = rng.choice((128, 128, 8, 1))
    c = max(lo, c // m * m)
    return c if c != 3072 else c + 8


def draw(rng):
    kind = rng.choice(("linear", "linear", "lineargrad", "moe", "score", "score", "scoregrad"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp16", "fp32"))
    if kind in ("linear", "lineargrad"):
        C = _width(rng, 64, 28672)
        R = _width(rng, 64, min(28672, 8192 * 28672 // C))
        cap = 16 if R * C > 1 << 26 else 64
        return dict(kind=kind, T=_log(rng, 1, cap), R=R, C=C, nbits=rng.choice((2, 3, 4, 4, 4, 5, 5, 8)),
                    groups=rng.choice(("channel", "channel", "128", "128", "64", "32", "order128")), dtype=dtype,
                    bias=kind == "linear" and rng.random() < 0.3) if R * C <= 1 << 26 else \
            dict(kind=kind, T=_log(rng, 1, cap), R=R, C=C, nbits=4, groups=rng.choice(("channel", "128")),
                 dtype=rng.choice(("bf16", "fp16")), bias=False)
    if kind == "moe":
        D, I = _width(rng, 256, 4096), _width(rng, 128, 7168)
        nbits = rng.choice((3, 4, 4, 5, 8))
        E = max(2, min(_log(rng, 4, 128), 1_000_000_000 // (D * I * nbits)))
        return dict(kind=kind, T=_log(rng, 1, 32), D=D, I=I, E=E, K=rng.randint(1, min(8, E)), nbits=nbits,
                    groups=rng.choice(("channel", "channel", "128", "128", "64", "order128")), dtype=dtype,
                    norm=rng.random() < 0.7)
    V = _log(rng, 500, 128256)
    N = _log(rng, 1, min(2048, 520_000_000 // (V * SIZES[dtype] * (2 if kind == "scoregrad" else 1))))
    return dict(kind=kind, N=N, V=V, top=0 if kind == "scoregrad" else rng.choice((0, 1, 5, 8, 20)), dtype=dtype,
                masked=rng.choice((0.0, 0.0, 0.3, 0.7)))


# --- inputs ------------------------------------------------------------------------------------


def _weight(gen, R, C, nbits, groups, batch=()):
    """A packed weight in export_packed's form: codes as a quantizer leaves them (near normal, the
    ends clipped), scales of a few per cent spread, and the group of every column."""
    size = C if groups == "channel" else int(groups.replace("order", ""))
    ng = -(-C // size)
    half = 1 << (nbits - 1)
    rows = math.prod(batch) * R
    words = (C * nbits + 31) // 32
    qweight = torch.empty((rows, words), dtype=torch.int32, device="cuda")
    blocks = -(-C // 32)
    for r0 in range(0, rows, 1 << 12):
        n = min(1 << 12, rows - r0)
        u = torch.randn((n, blocks * 32), generator=gen, device="cuda").mul_(half * 0.35).round_()
        u = u.clamp_(-half, half - 1).add_(half).to(torch.int32)
        u[:, C:] = 0
        u = u.view(n, blocks, 32)
        out = torch.zeros((n, blocks, nbits), dtype=torch.int32, device="cuda")
        for j in range(32):                      # 32 codes fill nbits words
            w, off = divmod(j * nbits, 32)
            out[:, :, w] |= u[:, :, j] << off
            if off + nbits > 32:
                out[:, :, w + 1] |= u[:, :, j] >> (32 - off)
        qweight[r0:r0 + n] = out.view(n, -1)[:, :words]
    scales = torch.rand((*batch, ng, R), generator=gen, device="cuda").add_(0.5).mul_(0.05 / half / math.sqrt(C / 1024))
    if groups.startswith("order"):
        order = torch.rand((*batch, C), generator=gen, device="cuda").argsort(-1)
        g_idx = (order.argsort(-1) // size).to(torch.int32)
    else:
        g_idx = (torch.arange(C, device="cuda") // size).to(torch.int32).expand(*batch, C).contiguous()
    entry = dict(qweight=qweight.view(*batch, R, words), scales=scales, g_idx=g_idx, nbits=nbits, bits=nbits, sym=True,
                 shape=(R, C), dtype="float16")
    if not groups.startswith("order"):
        entry["groupsize"] = size
    return entry


def _activations(gen, T, C, dtype):
    """Activations with a few outlier channels."""
    x = torch.randn((T, C), generator=gen, device="cuda")
    at = torch.randint(0, C, (min(8, C),), generator=gen, device="cuda")
    x[:, at] *= 20.0
    return x.to(DTYPES[dtype])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c, kind = case, case["kind"]
    s = dict(case=c, kind=kind)
    if kind == "linear":
        s["entry"] = _weight(gen, c["R"], c["C"], c["nbits"], c["groups"])
        s["x"] = _activations(gen, c["T"], c["C"], c["dtype"])
        s["bias"] = torch.randn(c["R"], generator=gen, device="cuda").to(DTYPES[c["dtype"]]) if c["bias"] else None
    elif kind == "lineargrad":
        s["entry"] = _weight(gen, c["R"], c["C"], c["nbits"], c["groups"])
        s["grad_y"] = torch.randn((c["T"], c["R"]), generator=gen, device="cuda").to(DTYPES[c["dtype"]])
    elif kind == "moe":
        s["gate"] = _weight(gen, c["I"], c["D"], c["nbits"], c["groups"], (c["E"],))
        s["up"] = _weight(gen, c["I"], c["D"], c["nbits"], c["groups"], (c["E"],))
        s["down"] = _weight(gen, c["D"], c["I"], c["nbits"], c["groups"], (c["E"],))
        s["router"] = (torch.randn((c["E"], c["D"]), generator=gen, device="cuda") / math.sqrt(c["D"])).to(DTYPES[c["dtype"]])
        s["x"] = _activations(gen, c["T"], c["D"], c["dtype"])
    else:
        N, V = c["N"], c["V"]
        z = torch.randn((N, V), generator=gen, device="cuda").mul_(3.0)
        s["targets"] = torch.randint(0, V, (N,), generator=gen, device="cuda")
        z.scatter_add_(1, s["targets"][:, None], 12.0 * torch.rand((N, 1), generator=gen, device="cuda"))
        if c["masked"]:
            drop = torch.rand((N, V), generator=gen, device="cuda") < c["masked"]
            z.masked_fill_(drop.scatter_(1, s["targets"][:, None], False), -math.inf)
            if N > 4:
                z[N // 2] = -math.inf                                # nothing is allowed
                z[N // 3, V // 2:] = torch.finfo(DTYPES[c["dtype"]]).min
                s["targets"][N // 3] %= V // 2
            s["targets"][torch.rand(N, generator=gen, device="cuda") < 0.1] = -100
        s["logits"] = z.to(DTYPES[c["dtype"]])
        if kind == "scoregrad":
            s["grad_logprob"] = torch.randn(N, generator=gen, device="cuda") / N
            s["grad_entropy"] = torch.randn(N, generator=gen, device="cuda") * (0.1 / N)
            # what the forward pass leaves: maximum, log of the sum, entropy of every row
            _, _, ls, H, _ = _scores(s["logits"])
            s["stats"] = torch.stack((s["logits"].float().amax(-1), ls, H), 1).contiguous()
    return s


# --- one pass ----------------------------------------------------------------------------------


def _dequant(entry):
    """The weight that a packed entry stands for, in 32 bits: [..., R, C]."""
    q, nb, C = entry["qweight"], entry["nbits"], entry["g_idx"].shape[-1]
    bit = torch.arange(C, device=q.device) * nb
    word, off = bit >> 5, bit & 31
    low = (q[..., word].to(torch.int64) & 0xFFFFFFFF) >> off
    high = q[..., (word + 1).clamp_max(q.shape[-1] - 1)].to(torch.int64) << (32 - off)
    codes = ((low | high) & ((1 << nb) - 1)) - (1 << (nb - 1))
    ng = entry["scales"].shape[-2]
    if ng == 1:
        return codes.float() * entry["scales"].transpose(-1, -2)
    at = entry["g_idx"].long()[..., None, :].expand(codes.shape)
    return codes.float() * entry["scales"].transpose(-1, -2).gather(-1, at)


def _scores(logits):
    """d = z - max, exp(d), log sum, entropy and which rows have anything left, in 32 bits."""
    z = logits.float()
    m = z.amax(-1)
    some = m > -math.inf
    m = torch.where(some, m, torch.zeros_like(m))
    d = z - m[:, None]
    e = d.exp()
    total = e.sum(-1)
    ls = torch.where(some, total, torch.ones_like(total)).log()
    H = torch.where(some, ls - torch.where(e > 0, e * d, torch.zeros_like(e)).sum(-1) / total, torch.zeros_like(ls))
    return d, e, ls, H, some


def _top(z, k):
    """The k largest of each row, equal values by their index: one key per value."""
    bits = (z.float() + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).to(torch.int64)
    key = (order << 32) - torch.arange(z.shape[-1], device=z.device)
    return key.topk(k, -1).indices


def run(state):
    kind = state["kind"]
    if own:
        import gptq_plus_mp_quant_amd as G
        if kind == "linear":
            return G.packed_linear(state["x"], state["entry"], bias=state["bias"])
        if kind == "lineargrad":
            return G.packed_linear_backward(state["grad_y"], state["entry"])
        if kind == "moe":
            c = state["case"]
            return G.packed_moe(state["x"], state["router"], state["gate"], state["up"], state["down"], c["K"],
                                norm_topk=c["norm"])
        if kind == "score":
            r = G.token_logprobs(state["logits"], state["targets"], top_k=state["case"]["top"])
            out = {"logprob": r.logprob, "entropy": r.entropy}
            return {**out, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs} if state["case"]["top"] else out
        return G.token_logprobs_backward(state["logits"], state["targets"], state["stats"], state["grad_logprob"],
                                         state["grad_entropy"])
    if kind == "linear":
        x = state["x"]
        y = x.float() @ _dequant(state["entry"]).t()
        if state["bias"] is not None:
            y = y + state["bias"].float()
        return y.to(x.dtype)
    if kind == "lineargrad":
        g = state["grad_y"]
        return (g.float() @ _dequant(state["entry"])).to(g.dtype)
    if kind == "moe":
        c, x = state["case"], state["x"].float()
        T, E, D, I = x.shape[0], c["E"], c["D"], c["I"]
        logits = x @ state["router"].float().t()
        ids = _top(logits, c["K"])
        p = logits.softmax(-1).gather(1, ids)
        if c["norm"]:
            p = p / p.sum(-1, keepdim=True)
        w = torch.zeros_like(logits).scatter(1, ids, p)
        # every expert on every token, the products of those not chosen weighted 0
        a = (x @ _dequant(state["gate"]).view(E * I, D).t()).view(T, E, I)
        b = (x @ _dequant(state["up"]).view(E * I, D).t()).view(T, E, I)
        h = (a * torch.sigmoid(a) * b * w[:, :, None]).view(T, E * I)
        y = h @ _dequant(state["down"]).transpose(1, 2).reshape(E * I, D)
        return y.to(state["x"].dtype)
    logits, targets = state["logits"], state["targets"]
    d, e, ls, H, some = _scores(logits)
    given = targets >= 0
    at = targets.clamp_min(0)[:, None]
    if kind == "score":
        lp = torch.where(some, d.gather(1, at)[:, 0] - ls, torch.full_like(ls, -math.inf))
        out = {"logprob": torch.where(given, lp, torch.zeros_like(lp)), "entropy": H}
        k = state["case"]["top"]
        if k:
            ids = _top(logits, k)
            out.update(top_ids=ids, top_logprobs=d.gather(1, ids) - ls[:, None])
        return out
    gl = torch.where(given, state["grad_logprob"], torch.zeros_like(ls))[:, None]
    gh = state["grad_entropy"][:, None]
    lp = d - ls[:, None]
    p = lp.exp()
    g = -torch.where(p > 0, p * (gl + gh * (lp + H[:, None])), torch.zeros_like(p))
    g = torch.where(some[:, None], g.scatter_add(1, at, gl), torch.zeros_like(g))
    return g.to(logits.dtype)


# --- what a pass cannot do without -------------------------------------------------------------


def _weight_bytes(R, C, nbits, groups):
    size = C if groups == "channel" else int(groups.replace("order", ""))
    return R * ((C * nbits + 31) // 32) * 4 + -(-C // size) * R * 4 + (4 * C if groups.startswith("order") else 0)


def work(case):
    c, e = case, SIZES[case["dtype"]]
    if c["kind"] in ("linear", "lineargrad"):
        T, R, C = c["T"], c["R"], c["C"]
        return {"bytes": _weight_bytes(R, C, c["nbits"], c["groups"]) + T * (R + C) * e + (R * e if c["bias"] else 0),
                "flops": 2 * T * R * C}
    if c["kind"] == "moe":
        T, D, I, E, K = c["T"], c["D"], c["I"], c["E"], c["K"]
        active = E * (1.0 - (1.0 - K / E) ** T)      # experts that T tokens choose between them
        one = 2 * _weight_bytes(I, D, c["nbits"], c["groups"]) + _weight_bytes(D, I, c["nbits"], c["groups"])
        return {"bytes": active * one + (E * D + 2 * T * D) * e, "flops": 2 * T * D * (E + 3 * K * I)}
    N, V = c["N"], c["V"]
    if c["kind"] == "score":
        return {"bytes": N * V * e + N * (8 + 8 + 12 * c["top"]), "flops": 6 * N * V}
    return {"bytes": 2 * N * V * e + N * 28, "flops": 8 * N * V}


# --- the same in 64 bits -----------------------------------------------------------------------


def _rows64(qweight, scales, g_idx, nbits):
    """One weight [R, C] in float64, from the bits of each row."""
    R, words = qweight.shape
    C = g_idx.numel()
    shifts = torch.arange(32, device=qweight.device, dtype=torch.int32)
    out = torch.empty((R, C), dtype=torch.float64, device=qweight.device)
    powers = 2.0 ** torch.arange(nbits, device=qweight.device, dtype=torch.float32)
    for r0 in range(0, R, 512):
        bits = (qweight[r0:r0 + 512, :, None] >> shifts) & 1
        field = bits.view(bits.shape[0], words * 32)[:, :C * nbits].reshape(-1, C, nbits).float() @ powers
        out[r0:r0 + 512] = (field.double() - 2.0 ** (nbits - 1)) * scales[:, r0:r0 + 512].double()[g_idx.long()].t()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("linear", "lineargrad"):
        t = s["entry"]
        W = _rows64(t["qweight"], t["scales"], t["g_idx"], t["nbits"])
        if kind == "lineargrad":
            return torch.mm(s["grad_y"].double(), W)
        y = torch.mm(s["x"].double(), W.t())
        return y if s["bias"] is None else y + s["bias"].double()
    if kind == "moe":
        x = s["x"].double()
        route = torch.mm(x, s["router"].double().t())
        y = torch.zeros((case["T"], case["D"]), dtype=torch.float64, device=x.device)
        best, ids = route.sort(dim=-1, descending=True, stable=True)
        p = torch.exp(best - route.logsumexp(-1, keepdim=True))[:, :case["K"]]
        if case["norm"]:
            p = p / p.sum(-1, keepdim=True)
        for ex in ids[:, :case["K"]].unique().tolist():
            W = [_rows64(s[n]["qweight"][ex], s[n]["scales"][ex], s[n]["g_idx"][ex], case["nbits"])
                 for n in ("gate", "up", "down")]
            t, k = (ids[:, :case["K"]] == ex).nonzero(as_tuple=True)
            a = torch.mm(x[t], W[0].t())
            y[t] += torch.mm(a / (1.0 + torch.exp(-a)) * torch.mm(x[t], W[1].t()), W[2].t()) * p[t, k][:, None]
        return y
    parts = []
    for n in range(0, case["N"], 64):
        z = s["logits"][n:n + 64].double()
        t = s["targets"][n:n + 64]
        empty = torch.isinf(z).all(-1)
        lp = torch.log_softmax(z, -1)
        plogp = torch.special.entr(lp.exp())                           # -p log p, 0 where p is 0
        H = torch.where(empty, 0.0, plogp.sum(-1))
        given = t >= 0
        if kind == "score":
            mine = torch.where(empty, -math.inf, lp[torch.arange(len(t), device=z.device), t.clamp_min(0)])
            top = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
            lt = torch.where(empty[:, None], -math.inf, lp.gather(1, top))
            parts.append((torch.where(given, mine, 0.0), H, top, lt))
        else:
            gl = s["grad_logprob"][n:n + 64].double() * given
            g = torch.zeros_like(z)
            g[torch.arange(len(t), device=z.device), t.clamp_min(0)] = gl
            gh = s["grad_entropy"][n:n + 64].double()[:, None]
            g = g - lp.exp() * gl[:, None] + gh * (plogp - lp.exp() * H[:, None])
            parts.append((torch.where(empty[:, None], 0.0, g),))
    whole = [torch.cat(p) for p in zip(*parts)]
    if kind == "scoregrad":
        return whole[0]
    out = {"logprob": whole[0], "entropy": whole[1]}
    return {**out, "top_ids": whole[2], "top_logprobs": whole[3]} if case["top"] else out
