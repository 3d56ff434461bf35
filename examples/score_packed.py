"""Quantise the linears of a small mixture-of-experts block, pack them, and answer from the packed form.

Eight experts (gate, up, down) and the output head are quantised to 4 bits in groups of 128 on random
calibration tokens, exported, stacked and run: ``packed_moe`` -> ``packed_linear`` -> ``token_logprobs``, for the
tokens of a prompt and then one token at a time, and the gradient of the score with respect to the head's
input.  The same is computed from the dequantized weights with torch, and the differences are printed.

    python examples/score_packed.py [--tokens 16] [--width 256] [--vocab 1000]
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import gptq_plus_mp_quant_amd as G  # noqa: E402


def quantise(weight, calibration, groupsize=128, bits=4):
    """The packed entry of one linear."""
    layer = torch.nn.Linear(weight.shape[1], weight.shape[0], bias=False, dtype=weight.dtype, device=weight.device)
    layer.weight.data.copy_(weight)
    gptq = G.GPTQ(layer)
    gptq.quantizer = G.WeightQuantizer()
    gptq.quantizer.configure(bits, perchannel=True, sym=True, mse=False)
    gptq.add_batch(calibration[None], None)
    gptq.fasterquant(percdamp=0.01, groupsize=groupsize)
    entry = G.export_packed(gptq)
    gptq.free()
    return entry


def run(tokens=16, width=256, inner=384, experts=8, top_k=2, vocab=1000, dtype=torch.bfloat16, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    calibration, wide = randn(512, width), randn(512, inner)
    shapes = dict(gate=(inner, width, calibration), up=(inner, width, calibration), down=(width, inner, wide))
    packed = {name: [quantise(randn(r, c, scale=c ** -0.5), x) for _ in range(experts)] for name, (r, c, x) in shapes.items()}
    head = quantise(randn(vocab, width, scale=width ** -0.5), calibration)
    stacked = {name: G.stack_packed(entries) for name, entries in packed.items()}
    router, x = randn(experts, width, scale=width ** -0.5), randn(tokens, width)
    targets = torch.randint(vocab, (tokens,), generator=gen, device="cuda")

    def answer(x, targets):
        h = x + G.packed_moe(x, router, stacked["gate"], stacked["up"], stacked["down"], top_k)
        return h, G.token_logprobs(G.packed_linear(h, head), targets, top_k=5)

    h, prompt = answer(x, targets)
    single = [answer(x[t:t + 1], targets[t:t + 1])[1] for t in range(tokens)]
    leaf = h.detach().requires_grad_()
    G.token_logprobs(G.packed_linear(leaf, head), targets).logprob.sum().backward()

    # the same with torch, in fp32, from the dequantized weights
    plain = {name: torch.stack([G.dequantize_packed(e).float() for e in entries]) for name, entries in packed.items()}
    xf = x.float()
    p = torch.softmax(xf @ router.float().t(), -1)
    weight, chosen = p.topk(top_k, -1)
    weight = weight / weight.sum(-1, keepdim=True)
    y = torch.zeros_like(xf)
    for t in range(tokens):
        for k in range(top_k):
            e = int(chosen[t, k])
            a = torch.nn.functional.silu(plain["gate"][e] @ xf[t]) * (plain["up"][e] @ xf[t])
            y[t] += weight[t, k] * (plain["down"][e] @ a)
    hf = (xf + y).requires_grad_()
    lp = torch.log_softmax(hf @ G.dequantize_packed(head).float().t(), -1).gather(1, targets[:, None])[:, 0]
    lp.sum().backward()
    lp = lp.detach()
    return dict(
        perplexity=float((-prompt.logprob).mean().exp()), plain_perplexity=float((-lp).mean().exp()),
        logprob_error=float((prompt.logprob - lp).abs().max()),
        single_error=float((torch.cat([s.logprob for s in single]) - prompt.logprob).abs().max()),
        gradient_error=float((leaf.grad.float() - hf.grad).norm() / hf.grad.norm()),
        best=prompt.top_ids[:, 0])


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=16)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--vocab", type=int, default=1000)
    a = ap.parse_args()
    r = run(tokens=a.tokens, width=a.width, vocab=a.vocab)
    print("perplexity %.3f (torch, from the dequantized weights: %.3f)" % (r["perplexity"], r["plain_perplexity"]))
    print("largest difference of a log probability: %.2e; of a token alone and in the prompt: %.2e"
          % (r["logprob_error"], r["single_error"]))
    print("relative difference of the gradient: %.2e" % r["gradient_error"])
