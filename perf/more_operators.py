"""Operators that adapt a packed model to its teacher, as cases that can be timed and checked.

A quantised model is packed once and stays as it is; what is lost is won back by low-rank adapters beside the
packed linears, trained on the full-precision model's most likely tokens, and many such adapters are served at
once over one packed model:

  lora         packed_linear_lora: a packed linear for tokens of several requests, each with its own adapter
               (or none): y = W x + b + s_a B_a (A_a x)
  loragrad     packed_linear_lora_backward: the gradients of x and of every adapter
  gated        packed_gated: act(Wg x) * (Wu x), the two packed projections, activation and product in one
  gatedgrad    packed_gated_backward: the gradient of x from the projections that the forward pass left
  distill      distillation_loss: the divergence from a teacher's top logits to the student's distribution
  distillgrad  distillation_loss_backward: the gradient of the student's logits

A case is a dict of plain values.  "groups" says how the scales of a weight lie: "channel" (one per row), a group
size (consecutive columns), or "order<size>" (groups of the act_order's permuted columns).  "ids" says whose tokens a
batch holds: "one" (one adapter for all), "mixed" (a request a token, some without an adapter), "runs" (prompts
one after another).
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # Serving, one token of one request over an attention projection, 8 adapters of rank 16 loaded: latency.
        dict(name="lora_token", kind="lora", T=1, R=4096, C=4096, r=16, n=8, ids="mixed", nbits=4, groups="128", dtype="bf16", bias=False),
        # A decoding step of 48 requests over an 8B model's gate projection, 16 adapters of rank 32 in any order.
        dict(name="lora_batch", kind="lora", T=48, R=14336, C=4096, r=32, n=16, ids="mixed", nbits=4, groups="128", dtype="bf16", bias=False),
        # No size a multiple of anything: fp32, w4 asymmetric along the act_order, rank 5, a handful of tokens.
        dict(name="loragrad_ragged", kind="loragrad", T=7, R=1026, C=1365, r=5, n=3, ids="mixed", nbits=5, groups="order128", dtype="fp32", bias=False),
        # A training step on a 128-token sample: one adapter of rank 64 beside an 8B model's down projection.
        dict(name="loragrad_train", kind="loragrad", T=128, R=4096, C=14336, r=64, n=1, ids="one", nbits=4, groups="128", dtype="bf16", bias=False),
        # Generation, one token: the first half of an 8B model's feed-forward block.
        dict(name="gated_token", kind="gated", T=1, I=14336, C=4096, nbits=4, groups="128", act="silu", dtype="bf16"),
        # The same of a 70B model for a batch of 24 sequences, w4 per channel: the largest weights.
        dict(name="gated_batch", kind="gated", T=24, I=28672, C=8192, nbits=4, groups="channel", act="silu", dtype="fp16"),
        # A small model's block of odd sizes in fp32, GELU, w4 asymmetric in groups of 64.
        dict(name="gatedgrad_short", kind="gatedgrad", T=5, I=2052, C=1000, nbits=5, groups="64", act="gelu_tanh", dtype="fp32"),
        # The gradient through an 8B model's block, 64 tokens.
        dict(name="gatedgrad_wide", kind="gatedgrad", T=64, I=14336, C=4096, nbits=4, groups="128", act="silu", dtype="bf16"),
        # A few answer tokens in fp32 with part of an odd vocabulary masked; the rest of the teacher's mass as one class.
        dict(name="distill_few", kind="distill", N=3, V=32003, K=20, tail="bucket", temperature=1.0, dtype="fp32", masked=0.3),
        # A calibration sample of 2048 tokens against the teacher's 64 best, softened.
        dict(name="distill_sample", kind="distill", N=2048, V=128256, K=64, tail="renormalise", temperature=2.0, dtype="bf16", masked=0.0),
        # The gradient for a dozen answers, fp32 logits.
        dict(name="distillgrad_few", kind="distillgrad", N=12, V=32003, K=16, tail="renormalise", temperature=1.0, dtype="fp32", masked=0.3),
        # The gradient of 1024 tokens of a sample, with the rest's class.
        dict(name="distillgrad_sample", kind="distillgrad", N=1024, V=128256, K=50, tail="bucket", temperature=1.0, dtype="bf16", masked=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width between lo and hi: a multiple of 128 or of 8 as model widths are, or any number."""
    c, m = _log(rng, lo, hi), rng.choice((128, 128, 8, 1))
    return max(lo, c // m * m)


def draw(rng):
    kind = rng.choice(("lora", "lora", "loragrad", "loragrad", "gated", "gated", "gatedgrad", "distill", "distill", "distillgrad"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp16", "fp32"))
    nbits, groups = rng.choice((2, 3, 4, 4, 4, 5, 5, 8)), rng.choice(("channel", "channel", "128", "128", "64", "32", "order128"))
    if kind in ("lora", "loragrad"):
        C = _width(rng, 64, 14336)
        R = _width(rng, 64, min(14336, (1 << 26) // C))
        ids = rng.choice(("one", "mixed", "mixed", "runs"))
        return dict(kind=kind, T=_log(rng, 1, 48 if R * C > 1 << 24 else 128), R=R, C=C, r=rng.choice((1, 4, 5, 8, 16, 16, 24, 32, 64, 100)),
                    n=1 if ids == "one" else _log(rng, 1, 32), ids=ids, nbits=nbits, groups=groups, dtype=dtype,
                    bias=kind == "lora" and rng.random() < 0.3)
    if kind in ("gated", "gatedgrad"):
        C = _width(rng, 64, 8192)
        return dict(kind=kind, T=_log(rng, 1, 64), I=_width(rng, 64, min(14336, (1 << 25) // C)), C=C, nbits=nbits, groups=groups,
                    act=rng.choice(("silu", "silu", "gelu", "gelu_tanh")), dtype=dtype)
    V = _log(rng, 500, 128256)
    N = _log(rng, 1, min(2048, 260_000_000 // (V * SIZES[dtype])))
    tail = rng.choice(("renormalise", "bucket"))
    return dict(kind=kind, N=N, V=V, K=_log(rng, 1, 200), tail=tail,
                temperature=1.0 if tail == "bucket" else rng.choice((0.7, 1.0, 1.0, 2.0, 4.0)), dtype=dtype, masked=rng.choice((0.0, 0.0, 0.3)))


# --- inputs ------------------------------------------------------------------------------------


def _weight(gen, R, C, nbits, groups):
    """A packed weight in export_packed's form: codes as a quantizer leaves them (near normal, the ends clipped),
    scales of a few per cent spread, and the group of every column."""
    size = C if groups == "channel" else int(groups.replace("order", ""))
    half, words, blocks = 1 << (nbits - 1), (C * nbits + 31) // 32, -(-C // 32)
    qweight = torch.empty((R, words), dtype=torch.int32, device="cuda")
    for r0 in range(0, R, 1 << 12):
        n = min(1 << 12, R - r0)
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
    scales = torch.rand((-(-C // size), R), generator=gen, device="cuda").add_(0.5).mul_(0.05 / half / math.sqrt(C / 1024))
    entry = dict(qweight=qweight, scales=scales, nbits=nbits, bits=nbits, sym=True, shape=(R, C), dtype="float16")
    if groups.startswith("order"):
        order = torch.rand(C, generator=gen, device="cuda").argsort()
        entry["g_idx"] = (order.argsort() // size).to(torch.int32)
    else:
        entry.update(g_idx=(torch.arange(C, device="cuda") // size).to(torch.int32), groupsize=size)
    return entry


def _activations(gen, T, C, dtype):
    """Activations with a few outlier channels."""
    x = torch.randn((T, C), generator=gen, device="cuda")
    at = torch.randint(0, C, (min(8, C),), generator=gen, device="cuda")
    x[:, at] *= 20.0
    return x.to(DTYPES[dtype])


def _whose(gen, T, n, ids):
    """The adapter of every token, -1 for none; None: the only adapter, for all."""
    if ids == "one":
        return None
    a = torch.randint(-1 if T > 1 else 0, n, (T,), generator=gen, device="cuda")
    return a.sort().values if ids == "runs" else a


def _teacher(gen, logits, K):
    """The K best tokens of a model near the student and their log probabilities, as token_logprobs gives them;
    some tokens have fewer, some (a prompt's) none: id -1."""
    N, V = logits.shape
    ids = torch.empty((N, K), dtype=torch.int64, device="cuda")
    lp = torch.empty((N, K), device="cuda")
    for n in range(0, N, 256):
        t = logits[n:n + 256].float()
        t = t + 0.7 * torch.randn(t.shape, generator=gen, device="cuda")
        best, at = t.topk(K, -1)
        ids[n:n + 256], lp[n:n + 256] = at, best - t.logsumexp(-1, keepdim=True)
    if N > 2:
        u = torch.rand((N, 1), generator=gen, device="cuda")
        ids[(u < 0.05) | ((u > 0.9) & (torch.arange(K, device="cuda") >= K // 2))] = -1
    return ids, lp


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c, kind = case, case["kind"]
    s = dict(case=c, kind=kind)
    if kind in ("lora", "loragrad"):
        T, R, C, r, n, dt = c["T"], c["R"], c["C"], c["r"], c["n"], DTYPES[c["dtype"]]
        s["entry"] = _weight(gen, R, C, c["nbits"], c["groups"])
        s["x"] = _activations(gen, T, C, c["dtype"])
        s["a"] = (torch.randn((n, r, C), generator=gen, device="cuda") / math.sqrt(C)).to(dt)
        s["b"] = (0.3 * torch.randn((n, R, r), generator=gen, device="cuda") / math.sqrt(r)).to(dt)
        s["scaling"] = torch.rand(n, generator=gen, device="cuda") + 0.5
        s["ids"] = _whose(gen, T, n, c["ids"])
        s["bias"] = torch.randn(R, generator=gen, device="cuda").to(dt) if c["bias"] else None
        if kind == "loragrad":
            s["grad_y"] = torch.randn((T, R), generator=gen, device="cuda").to(dt)
    elif kind in ("gated", "gatedgrad"):
        s["gate"] = _weight(gen, c["I"], c["C"], c["nbits"], c["groups"])
        s["up"] = _weight(gen, c["I"], c["C"], c["nbits"], c["groups"])
        x = _activations(gen, c["T"], c["C"], c["dtype"])
        if kind == "gated":
            s["x"] = x
        else:
            # what the forward pass leaves: both projections, fp32 [T, 2, I]
            s["pre"] = torch.stack([x.float() @ _dequant(s[k]).t() for k in ("gate", "up")], 1)
            s["grad_h"] = torch.randn((c["T"], c["I"]), generator=gen, device="cuda").to(DTYPES[c["dtype"]])
    else:
        N, V, K = c["N"], c["V"], min(c["K"], c["V"])
        z = torch.randn((N, V), generator=gen, device="cuda").mul_(3.0)
        likely = torch.randint(0, V, (N, 4), generator=gen, device="cuda")
        z.scatter_add_(1, likely, 12.0 * torch.rand((N, 4), generator=gen, device="cuda"))
        s["logits"] = z.to(DTYPES[c["dtype"]])
        s["teacher_ids"], s["teacher_logprobs"] = _teacher(gen, s["logits"], K)
        if c["masked"]:                          # tokens that a grammar rules out, none of the teacher's
            drop = torch.rand((N, V), generator=gen, device="cuda") < c["masked"]
            drop.scatter_(1, s["teacher_ids"].clamp_min(0), False)
            s["logits"].masked_fill_(drop, -math.inf)
            s["logits"][0].masked_fill_(drop[0], torch.finfo(DTYPES[c["dtype"]]).min)
        if kind == "distillgrad":
            s["grad_loss"] = torch.rand(N, generator=gen, device="cuda") / N
            s["stats"] = _distill(s)[1]
    return s


# --- one pass ----------------------------------------------------------------------------------


def _dequant(entry):
    """The weight that a packed entry stands for, in 32 bits: [R, C]."""
    q, nb, C = entry["qweight"], entry["nbits"], entry["g_idx"].numel()
    bit = torch.arange(C, device=q.device) * nb
    word, off = bit >> 5, bit & 31
    low = (q[:, word].to(torch.int64) & 0xFFFFFFFF) >> off
    high = q[:, (word + 1).clamp_max(q.shape[1] - 1)].to(torch.int64) << (32 - off)
    codes = ((low | high) & ((1 << nb) - 1)) - (1 << (nb - 1))
    return codes.float() * entry["scales"][entry["g_idx"].long()].t()


def _of_adapter(state):
    """For every adapter the mask of its tokens as a column of 0 and its scaling."""
    T, n = state["x"].shape[0], state["a"].shape[0]
    ids = state["ids"] if state["ids"] is not None else torch.zeros(T, dtype=torch.int64, device="cuda")
    return [(ids == i).float()[:, None] * state["scaling"][i] for i in range(n)]


def _act(name, a):
    """An activation and its derivative."""
    if name == "silu":
        s = 1.0 / (1.0 + (-a).exp())
        return a * s, s * (1.0 + a * (1.0 - s))
    if name == "gelu":
        cdf = 0.5 * torch.erfc(a * -math.sqrt(0.5))
        return a * cdf, cdf + a * (-0.5 * a * a).exp() / math.sqrt(2.0 * math.pi)
    k = 2.0 * math.sqrt(2.0 / math.pi)
    s = 1.0 / (1.0 + (-k * (a + 0.044715 * a * a * a)).exp())
    return a * s, s + a * s * (1.0 - s) * k * (1.0 + 3.0 * 0.044715 * a * a)


def _distill(state):
    """The loss of every row and what its gradient needs, [N, 8]: maximum and log of the sum of the exponents over all
    logits, the same over those outside the teacher's list (over all where there is no class for the rest), the teacher's
    maximum and log sum, its whole mass, and the factor of the rest's probabilities in the gradient.  Sums next to 1 and
    their logarithms are taken in 64 bits."""
    c, logits = state["case"], state["logits"]
    inv, bucket = 1.0 / c["temperature"], c["tail"] == "bucket"
    ids, t = state["teacher_ids"], state["teacher_logprobs"].double()
    used, at = ids >= 0, ids.clamp_min(0)
    z = logits.float()

    def log_sum(v):
        m = v.amax(-1)
        m = torch.where(m > -math.inf, m, torch.zeros_like(m))
        s = ((v - m[:, None]) * inv).exp().sum(-1, dtype=torch.float64)
        return m, s.log()

    m, ls = log_sum(z)
    mine = (z.gather(1, at) - m[:, None]).double() * inv - ls[:, None]
    if bucket:
        rest = torch.ones_like(z, dtype=torch.bool)
        row = torch.arange(z.shape[0], device=z.device)[:, None].expand(at.shape)
        rest[row[used], at[used]] = False
        mr, lr = log_sum(torch.where(rest, z, torch.full_like(z, -math.inf)))
        mt, lt = torch.zeros_like(ls), torch.zeros_like(ls)
    else:
        mr, lr = m, ls
        mt = torch.where(used, t, torch.full_like(t, -math.inf)).amax(-1)
        mt = torch.where(mt > -math.inf, mt, torch.zeros_like(mt))
        lt = torch.where(used, ((t - mt[:, None]) * inv).exp(), torch.zeros_like(t)).sum(-1).log()
    logp = (t - mt[:, None]) * inv - lt[:, None]
    p = torch.where(used, logp.exp(), torch.zeros_like(logp))
    mass = p.sum(-1)
    loss = torch.where(p > 0, p * (logp - mine), torch.zeros_like(p)).sum(-1)
    factor = mass
    if bucket:
        r = (1.0 - mass).clamp_min(0.0)
        log_rest = (mr - m).double() + lr - ls
        loss = loss + torch.where(r > 0, r * (r.log() - log_rest), torch.zeros_like(r))
        mass = mass + r
        factor = log_rest.exp() * mass - r
    some = used.any(-1)
    loss = torch.where(some, loss, torch.zeros_like(loss))
    mass = torch.where(some, mass, torch.zeros_like(mass))
    factor = torch.where(some, factor, torch.zeros_like(factor))
    stats = torch.stack([v.double() for v in (m, ls, mr, lr, mt, lt, mass, factor)], 1)
    return loss.float(), stats.float(), p


def run(state):
    kind, c = state["kind"], state["case"]
    if own:
        import gptq_plus_mp_quant_amd as G
        if kind == "lora":
            return G.packed_linear_lora(state["x"], state["entry"], state["a"], state["b"], state["ids"], state["scaling"],
                                        bias=state["bias"])
        if kind == "loragrad":
            gx, ga, gb = G.packed_linear_lora_backward(state["grad_y"], state["x"], state["entry"], state["a"], state["b"],
                                                       state["ids"], state["scaling"])
            return {"grad_x": gx, "grad_a": ga, "grad_b": gb}
        if kind == "gated":
            return G.packed_gated(state["x"], state["gate"], state["up"], activation=c["act"])
        if kind == "gatedgrad":
            return G.packed_gated_backward(state["grad_h"], state["pre"], state["gate"], state["up"], activation=c["act"])
        if kind == "distill":
            return G.distillation_loss(state["logits"], state["teacher_ids"], state["teacher_logprobs"],
                                       temperature=c["temperature"], tail=c["tail"]).loss
        return G.distillation_loss_backward(state["logits"], state["teacher_ids"], state["teacher_logprobs"], state["stats"],
                                            state["grad_loss"], temperature=c["temperature"], tail=c["tail"])
    if kind in ("lora", "loragrad"):
        x, W, dt = state["x"].float(), _dequant(state["entry"]), state["x"].dtype
        A, B = state["a"].float(), state["b"].float()
        masks = _of_adapter(state)
        if kind == "lora":
            y = x @ W.t()
            for m, a, b in zip(masks, A, B):
                y = y + m * ((x @ a.t()) @ b.t())
            return (y if state["bias"] is None else y + state["bias"].float()).to(dt)
        g = state["grad_y"].float()
        gx, ga, gb = g @ W, [], []
        for m, a, b in zip(masks, A, B):
            v, u = m * (g @ b), m * (x @ a.t())
            gx = gx + v @ a
            ga.append(v.t() @ x)
            gb.append(g.t() @ u)
        return {"grad_x": gx.to(dt), "grad_a": torch.stack(ga).to(dt), "grad_b": torch.stack(gb).to(dt)}
    if kind == "gated":
        x = state["x"].float()
        return (_act(c["act"], x @ _dequant(state["gate"]).t())[0] * (x @ _dequant(state["up"]).t())).to(state["x"].dtype)
    if kind == "gatedgrad":
        g, (a, b) = state["grad_h"].float(), state["pre"].unbind(1)
        f, df = _act(c["act"], a)
        return ((g * b * df) @ _dequant(state["gate"]) + (g * f) @ _dequant(state["up"])).to(state["grad_h"].dtype)
    loss, stats, p = _distill(state)
    if kind == "distill":
        return loss
    logits, ids = state["logits"], state["teacher_ids"]
    m, ls, mr, lr, _, _, mass, factor = state["stats"].unbind(1)
    inv = 1.0 / c["temperature"]
    z = logits.float()
    g = (((z - mr[:, None]) * inv - lr[:, None]).clamp_max(0.0)).exp() * factor[:, None]
    at = ids.clamp_min(0)
    mine = ((z.gather(1, at) - m[:, None]) * inv - ls[:, None]).exp() * mass[:, None] - p.float()
    row = torch.arange(z.shape[0], device=z.device)[:, None].expand(at.shape)
    g[row[ids >= 0], at[ids >= 0]] = mine[ids >= 0]
    return (g * (state["grad_loss"] * inv)[:, None]).to(logits.dtype)


# --- what a pass cannot do without -------------------------------------------------------------


def _weight_bytes(R, C, nbits, groups):
    size = C if groups == "channel" else int(groups.replace("order", ""))
    return R * ((C * nbits + 31) // 32) * 4 + -(-C // size) * R * 4 + (4 * C if groups.startswith("order") else 0)


def work(case):
    c, e = case, SIZES[case["dtype"]]
    if c["kind"] in ("lora", "loragrad"):
        T, R, C, r, n = c["T"], c["R"], c["C"], c["r"], c["n"]
        active = n * (1.0 - (1.0 - 1.0 / n) ** T) if n > 1 else 1      # adapters that T tokens have between them
        pair = r * (R + C) * e
        w = _weight_bytes(R, C, c["nbits"], c["groups"])
        if c["kind"] == "lora":
            return {"bytes": w + T * (R + C) * e + active * pair + (R * e if c["bias"] else 0) + 12 * T,
                    "flops": 2 * T * R * C + 2 * T * r * (R + C)}
        return {"bytes": w + T * (R + 2 * C) * e + (active + n) * pair + 12 * T, "flops": 2 * T * R * C + 8 * T * r * (R + C)}
    if c["kind"] in ("gated", "gatedgrad"):
        T, I, C = c["T"], c["I"], c["C"]
        return {"bytes": 2 * _weight_bytes(I, C, c["nbits"], c["groups"]) + T * (I + C) * e + (8 * T * I if c["kind"] == "gatedgrad" else 0),
                "flops": 4 * T * I * C}
    N, V, K = c["N"], c["V"], min(c["K"], c["V"])
    if c["kind"] == "distill":
        return {"bytes": N * V * e + N * (12 * K + 4), "flops": 4 * N * V}
    return {"bytes": 2 * N * V * e + N * (12 * K + 36), "flops": 5 * N * V}


# --- the same in 64 bits -----------------------------------------------------------------------


def _rows64(entry):
    """A weight [R, C] in float64, from the bits of each row."""
    qweight, scales, nbits, group = entry["qweight"], entry["scales"], entry["nbits"], entry["g_idx"].long()
    R, words = qweight.shape
    C = group.numel()
    shifts = torch.arange(32, device=qweight.device, dtype=torch.int32)
    powers = 2.0 ** torch.arange(nbits, device=qweight.device, dtype=torch.float32)
    out = torch.empty((R, C), dtype=torch.float64, device=qweight.device)
    for r0 in range(0, R, 512):
        bits = (qweight[r0:r0 + 512, :, None] >> shifts) & 1
        field = bits.view(bits.shape[0], words * 32)[:, :C * nbits].reshape(-1, C, nbits).float() @ powers
        out[r0:r0 + 512] = (field.double() - 2.0 ** (nbits - 1)) * scales[:, r0:r0 + 512].double()[group].t()
    return out


def _activation64(name, a):
    """Value and derivative by differentiation."""
    a = a.detach().requires_grad_()
    with torch.enable_grad():
        if name == "silu":
            f = a * torch.sigmoid(a)
        elif name == "gelu":
            f = a * torch.special.ndtr(a)
        else:
            f = 0.5 * a * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (a + 0.044715 * a.pow(3))))
        (df,) = torch.autograd.grad(f.sum(), a)
    return f.detach(), df


def _classes64(s, case, n0, n1):
    """Of rows n0..n1: log probabilities of the student over its tokens, and the teacher's probabilities by token."""
    z = s["logits"][n0:n1].double() / case["temperature"]
    ids, t = s["teacher_ids"][n0:n1], s["teacher_logprobs"][n0:n1].double()
    lq = torch.log_softmax(z, -1)
    t = torch.where(ids >= 0, t, -math.inf)
    p = torch.softmax(t / case["temperature"], -1) if case["tail"] == "renormalise" else t.exp()
    p = torch.where(ids >= 0, p, 0.0)
    full = torch.zeros_like(lq).scatter_add_(1, ids.clamp_min(0), p)
    return lq, full, (ids >= 0).any(-1), ids


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("lora", "loragrad"):
        W, x = _rows64(s["entry"]), s["x"].double()
        T, n = case["T"], case["n"]
        ids = s["ids"].tolist() if s["ids"] is not None else [0] * T
        A, B, scaling = s["a"].double(), s["b"].double(), s["scaling"].double()
        if kind == "lora":
            y = torch.mm(x, W.t())
            if s["bias"] is not None:
                y += s["bias"].double()
            for t, i in enumerate(ids):
                if i >= 0:
                    y[t] += scaling[i] * torch.mv(B[i], torch.mv(A[i], x[t]))
            return y
        g = s["grad_y"].double()
        gx, ga, gb = torch.mm(g, W), torch.zeros_like(A), torch.zeros_like(B)
        for i in range(n):
            of = torch.tensor([t for t in range(T) if ids[t] == i], dtype=torch.int64, device=x.device)
            back = scaling[i] * torch.mm(g[of], B[i])
            gx[of] += torch.mm(back, A[i])
            ga[i] = torch.mm(back.t().contiguous(), x[of])
            gb[i] = scaling[i] * torch.mm(g[of].t().contiguous(), torch.mm(x[of], A[i].t()))
        return {"grad_x": gx, "grad_a": ga, "grad_b": gb}
    if kind == "gated":
        x = s["x"].double()
        f, _ = _activation64(case["act"], torch.mm(x, _rows64(s["gate"]).t()))
        return f * torch.mm(x, _rows64(s["up"]).t())
    if kind == "gatedgrad":
        g, pre = s["grad_h"].double(), s["pre"].double()
        f, df = _activation64(case["act"], pre[:, 0])
        return torch.mm(g * pre[:, 1] * df, _rows64(s["gate"])) + torch.mm(g * f, _rows64(s["up"]))
    parts = []
    for n in range(0, case["N"], 64):
        lq, p, some, ids = _classes64(s, case, n, n + 64)
        listed_ = torch.zeros_like(p, dtype=torch.bool)
        for k in range(ids.shape[1]):
            listed_[torch.arange(len(ids), device=ids.device), ids[:, k].clamp_min(0)] |= ids[:, k] >= 0
        r = (1.0 - p.sum(-1)).clamp_min(0.0) if case["tail"] == "bucket" else torch.zeros_like(p[:, 0])
        lr = torch.where(listed_, -math.inf, lq).logsumexp(-1)
        if kind == "distill":
            loss = torch.where(p > 0, torch.xlogy(p, p) - p * lq, 0.0).sum(-1)
            loss = loss + torch.where(r > 0, torch.xlogy(r, r) - r * lr, 0.0)
            parts.append(torch.where(some, loss, 0.0))
        else:
            g = lq.exp() * (p.sum(-1) + r)[:, None] - p
            g = g - torch.where(listed_ | torch.isinf(lq), 0.0, r[:, None] * (lq - lr[:, None]).exp())
            g = torch.where(some[:, None], g, 0.0)
            parts.append(g * s["grad_loss"][n:n + 64].double()[:, None] / case["temperature"])
    return torch.cat(parts)
