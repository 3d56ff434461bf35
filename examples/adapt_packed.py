"""Train low-rank adapters on a packed feed-forward block and output head against the full-precision model's most
likely tokens, then answer with two requests' adapters at once.

The linears (gate, up, down, head) are quantised to 4 bits in groups of 128 on random calibration tokens and packed.
The full-precision model's best tokens come from ``token_logprobs``; a step is ``packed_gated`` ->
``packed_linear_lora`` (down) -> ``packed_linear_lora`` (head) -> ``distillation_loss`` and its gradients.  The first
step's loss and gradients are computed in fp64 from the dequantized weights as well, and the differences are printed.

    python examples/adapt_packed.py [--tokens 64] [--width 256] [--vocab 1000] [--rank 8] [--steps 20]
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
sys.path.insert(0, str(Path(__file__).resolve().parent))
import gptq_plus_mp_quant_amd as G  # noqa: E402
from score_packed import quantise  # noqa: E402


def run(tokens=64, width=256, inner=512, vocab=1000, rank=8, steps=20, top_k=20, tail="bucket", dtype=torch.bfloat16, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    shapes = dict(gate=(inner, width), up=(inner, width), down=(width, inner), head=(vocab, width))
    weights = {name: randn(r, c, scale=(4 if name == "head" else 1) * c ** -0.5) for name, (r, c) in shapes.items()}
    packed = {name: quantise(w, randn(512, w.shape[1])) for name, w in weights.items()}
    x = randn(tokens, width)

    def block(x, w):
        h = torch.nn.functional.silu(x @ w["gate"].t()) * (x @ w["up"].t())
        return x + h @ w["down"].t()

    # the teacher: the full-precision weights; what is kept of it is a few numbers a token
    teacher = {name: w.float() for name, w in weights.items()}
    logits = block(x.float(), teacher) @ teacher["head"].t()
    kept = G.token_logprobs(logits, torch.zeros(tokens, dtype=torch.int64, device="cuda"), top_k=top_k)

    adapters = {}
    for name in ("down", "head"):
        r, c = shapes[name]
        adapters[name] = [randn(1, rank, c, scale=c ** -0.5).float().requires_grad_(), randn(1, r, rank, scale=0.02).float().requires_grad_()]
    leaves = [t for pair in adapters.values() for t in pair]

    def student(x, adapters, ids=None):
        adapters = {name: [t.to(dtype) for t in pair] for name, pair in adapters.items()}       # kept in fp32
        h = G.packed_gated(x, packed["gate"], packed["up"])
        h = x + G.packed_linear_lora(h, packed["down"], *adapters["down"], ids, 2.0)
        return G.packed_linear_lora(h, packed["head"], *adapters["head"], ids, 2.0)

    def loss_of(logits):
        return G.distillation_loss(logits, kept.top_ids, kept.top_logprobs, tail=tail).loss.mean()

    first = loss_of(student(x, adapters))
    first.backward()

    # the same in fp64 from the dequantized weights
    plain = {name: G.dequantize_packed(e).double() for name, e in packed.items()}
    twins = {name: [t.detach().double()[0].requires_grad_() for t in pair] for name, pair in adapters.items()}
    xd = x.double()
    h = torch.nn.functional.silu(xd @ plain["gate"].t()) * (xd @ plain["up"].t())
    h = xd + h @ plain["down"].t() + 2.0 * (h @ twins["down"][0].t()) @ twins["down"][1].t()
    z = h @ plain["head"].t() + 2.0 * (h @ twins["head"][0].t()) @ twins["head"][1].t()
    lq, logp = torch.log_softmax(z, -1), kept.top_logprobs.double()
    if tail == "renormalise":
        logp = torch.log_softmax(logp, -1)
    p = logp.exp()
    want = (p * (logp - lq.gather(1, kept.top_ids))).sum(-1)
    if tail == "bucket":
        rest = 1.0 - p.sum(-1)
        others = torch.logsumexp(lq.scatter(1, kept.top_ids, -torch.inf), -1)
        want = want + rest * (rest.log() - others)
    want = want.mean()
    want.backward()
    # the logits' gradient is a difference of probabilities: how much larger its terms are
    q, full = lq.detach().exp(), torch.zeros_like(lq).scatter(1, kept.top_ids, p)
    terms = float((q + full).norm() / (q - full).norm())
    errors = [float((t.grad.double()[0] - u.grad).norm() / u.grad.norm())
              for pair, twin in zip(adapters.values(), twins.values()) for t, u in zip(pair, twin)]

    optimizer = torch.optim.Adam(leaves, lr=2e-3)
    losses = [float(first.detach())]
    for _ in range(steps):
        optimizer.step()
        optimizer.zero_grad()
        loss = loss_of(student(x, adapters))
        loss.backward()
        losses.append(float(loss.detach()))

    # serving: this adapter and a second one, every other token with the second, the last token with none
    with torch.no_grad():
        two = {name: [torch.cat([t, 0.5 * t]) for t in pair] for name, pair in adapters.items()}
        ids = torch.arange(tokens, device="cuda") % 2
        ids[-1] = -1
        served = student(x, two, ids)
        alone = torch.cat([student(x[t:t + 1], {n: [a[i:i + 1] for a in pair] for n, pair in two.items()} if i >= 0 else two,
                                   None if i >= 0 else ids[t:t + 1]) for t, i in enumerate(ids.tolist())])
        serving_error = float((served.double() - alone.double()).norm() / alone.double().norm())
    return dict(loss=losses[0], plain_loss=float(want.detach()), gradient_errors=errors, terms=terms, losses=losses,
                serving_error=serving_error)


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    for name, default in (("tokens", 64), ("width", 256), ("vocab", 1000), ("rank", 8), ("steps", 20)):
        parser.add_argument(f"--{name}", type=int, default=default)
    for key, value in run(**vars(parser.parse_args())).items():
        print(f"{key}: {value}")
