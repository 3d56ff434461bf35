"""distillation_loss and its gradient against the definitions in 64 bits.

Bounds, in units of 2^-24: a term exp(d) of a sum is off by a few units and |d| more (d, its product and the power are
rounded), so the log of a row's sum is off by 64 + sqrt(V) (the lanes' fp32 sums; the |d| are weighted by exp(d)).
The loss is the teacher's probabilities times such logarithms, all else of it 64 bits, rounded once.  A probability in the
gradient is off by 64 + sqrt(V) + 4 |log p| of itself, and by 2^-126, below which it may be 0."""
import math

import numpy as np
import pytest
import torch

from gptq_plus_mp_quant_amd import distillation_loss, distillation_loss_backward, token_logprobs
from tests._packed import ROUND, TINY, assert_within
from tests._util import rng

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF = math.inf
U = 2.0 ** -24
TAILS = [("renormalise", 1.0), ("renormalise", 2.5), ("bucket", 1.0)]


def randn(seed, *shape, dtype=F32, scale=1.0):
    return (torch.from_numpy(rng(seed).standard_normal(shape, dtype=np.float32)) * scale).to(dtype)


def teacher(seed, z, k, noise=0.7):
    """The k best of a model near z, as token_logprobs leaves them."""
    t = z.float() + randn(seed, *z.shape, scale=noise)
    best, ids = t.topk(k, -1)
    return ids, (best - t.logsumexp(-1, keepdim=True)).float()


def definition(z, ids, t, temperature, tail):
    """loss, the gradient for a gradient of 1, and the bounds of both, in float64."""
    z, t = z.double() / temperature, t.double()
    N, V = z.shape
    unit = (64 + math.sqrt(V)) * U
    used, at = ids >= 0, ids.clamp(0, V - 1)
    empty = (z == -INF).all(-1)
    lq = torch.where(empty[:, None], -INF, z - torch.where(empty, 0.0, z.logsumexp(-1))[:, None])
    t = torch.where(used, t, -INF)
    p = t.exp() if tail == "bucket" else torch.where((t == -INF).all(-1, keepdim=True), 0.0, torch.softmax(t / temperature, -1))
    p = torch.where(used, p, 0.0)
    logp = torch.where(p > 0, p.log(), 0.0)
    mine = lq.gather(1, at)
    loss = torch.where(p > 0, p * (logp - mine), 0.0).sum(-1)
    mass = p.sum(-1)
    off = unit * mass
    full = torch.zeros_like(z).scatter_add_(1, at, p)
    listed = torch.zeros_like(z).scatter_add_(1, at, used.double()) > 0
    q = lq.exp()
    wide = 4 * torch.where(lq > -INF, lq.abs(), 0.0) * U
    if tail == "bucket":
        rest = torch.where(listed, -INF, lq)
        none = (rest == -INF).all(-1)
        lrest = torch.where(none, -INF, rest.logsumexp(-1))
        r = (1.0 - mass).clamp_min(0.0)
        r = torch.where(none & (r <= 2.0 ** -20), 0.0, r)
        loss = loss + torch.where(r > 0, r * (torch.where(r > 0, r, 1.0).log() - lrest), 0.0)
        off = off + 2 * unit * r
        mass = mass + r
        w = torch.where(listed | (rest == -INF), 0.0, (rest - torch.where(none, 0.0, lrest)[:, None]).exp())
        grad = torch.where(listed, q * mass[:, None] - full, w * (lrest.exp() * mass - r)[:, None])
        size = torch.where(listed, q * mass[:, None] + full, w * (lrest.exp() * mass + r)[:, None])
    else:
        grad, size = q * mass[:, None] - full, q * mass[:, None] + full
    wide = wide + 4 * U * torch.where(full > 0, full.log().abs(), 0.0)
    if tail == "bucket":
        wide = wide + 4 * U * torch.where(w > 0, w.log().abs(), 0.0)
    bound = (unit + wide) * size + 2.0 ** -126 * (1 + mass[:, None])
    some = used.any(-1)
    loss, off = torch.where(some, loss, 0.0), torch.where(some, off, 0.0)
    dead = empty | ~some
    grad, bound = torch.where(dead[:, None], 0.0, grad) / temperature, torch.where(dead[:, None], 0.0, bound) / temperature
    bad = (ids >= V).any(-1) | torch.isnan(z).any(-1) | (z == INF).any(-1)
    bad = some & bad
    loss, grad = torch.where(bad, torch.nan, loss), torch.where(bad[:, None], torch.nan, grad)
    return loss, off + U * loss.abs(), grad, bound


def check(z, ids, t, temperature=1.0, tail="renormalise", z_dev=None, grad=True):
    zd = z.to(DEV) if z_dev is None else z_dev
    args = zd, ids.to(DEV), t.to(DEV)
    r = distillation_loss(*args, temperature, tail)
    loss, off, g, bound = definition(z, ids, t, temperature, tail)
    assert r.loss.dtype == F32 and r.loss.shape == z.shape[:-1]
    assert_within(r.loss, loss, off, "loss")
    if not grad:
        return r, None
    gl = randn(91, z.shape[0])
    got = distillation_loss_backward(*args, r.stats, gl.to(DEV), temperature, tail)
    assert got.dtype == z.dtype and got.shape == z.shape
    want, size = g * gl.double()[:, None], gl.double().abs()[:, None]
    assert_within(got, want, bound * size + (ROUND[z.dtype] + 2 * U) * want.abs() + TINY[z.dtype] + 2.0 ** -126, "gradient")
    return r, got


@pytest.mark.parametrize("tail,temperature", TAILS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("N,V,k", [(1, 1, 1), (1, 2, 2), (2, 3, 1), (3, 63, 20), (1, 64, 64), (4, 65, 64), (5, 500, 256), (1, 32003, 20),
                                   (7, 8191, 8), (2, 8193, 1), (300, 257, 4), (17, 32000, 100), (1, 128256, 64), (3, 100001, 20),
                                   (520, 4100, 9), (2, 300001, 50)])
def test_shapes(N, V, k, dtype, tail, temperature):
    z = randn(N + V, N, V, dtype=dtype, scale=3.0)
    check(z, *teacher(V, z, k), temperature, tail)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("tail,temperature", TAILS)
@pytest.mark.parametrize("N,V", [(6, 50), (6, 8199), (515, 4099)])
def test_masks(N, V, tail, temperature, dtype):
    """-inf, the type's lowest value and most of a row masked, none of the teacher's tokens; then some of them too."""
    z = randn(1, N, V, dtype=dtype, scale=2.0)
    ids, t = teacher(2, z, 7)
    for row, (value, share) in enumerate(((-INF, 0.3), (torch.finfo(dtype).min, 0.3), (-INF, 0.99), (torch.finfo(dtype).min, 0.99),
                                          (-INF, 1.0), (torch.finfo(dtype).min, 1.0))):
        drop = torch.from_numpy(rng(row).random(V) < share)
        drop[ids[row]] = False
        z[row, drop] = value
    check(z, ids, t, temperature, tail)
    z[0, ids[0, 2]] = -INF                       # the student rules out what the teacher would say
    z[1, ids[1, 0]] = torch.finfo(dtype).min
    r, _ = check(z, ids, t, temperature, tail)
    assert float(r.loss[0]) == INF
    t[0, 2] = -INF                               # the teacher too
    r, _ = check(z, ids, t, temperature, tail)
    assert math.isfinite(float(r.loss[0]))


@pytest.mark.parametrize("tail,temperature", TAILS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("N,V", [(9, 40), (9, 8199), (520, 4099)])
def test_lists(N, V, tail, temperature, dtype):
    """Short lists, none, entries anywhere in any order, a list of the whole vocabulary, ids outside."""
    z = randn(3, N, V, dtype=dtype)
    ids, t = teacher(4, z, 33)
    mix = torch.from_numpy(rng(5).permutation(33))
    ids, t = ids[:, mix], t[:, mix]
    ids[1, 1:], ids[2, ::2], ids[3] = -1, -5, -1
    t[1, 1:], t[3] = float("nan"), INF           # what stands beside no entry is nothing
    ids[4, 32] = V                               # outside the vocabulary
    ids[5, 0] = 1 << 40
    r, g = check(z, ids, t, temperature, tail)
    loss = r.loss.cpu()
    assert float(loss[3]) == 0.0 and not bool(g[3].any()) and bool(torch.isnan(loss[4:6]).all()) and bool(torch.isnan(g[4:6]).all())


@pytest.mark.parametrize("tail,temperature", TAILS)
@pytest.mark.parametrize("N,V", [(4, 8199), (513, 4099)])
def test_the_same_token_twice(N, V, tail, temperature):
    """Its probabilities add up, as two terms of the sum."""
    z = randn(3, N, V)
    ids, t = teacher(4, z, 12)
    ids[:, 7], ids[0, 8], ids[1, 11] = ids[:, 2], ids[0, 2], ids[1, 0]
    t = t - math.log(2.0)
    check(z, ids, t, temperature, tail)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("tail,temperature", TAILS)
@pytest.mark.parametrize("N,V", [(6, 40), (6, 70001), (515, 5003)])
def test_non_finite_rows(N, V, tail, temperature, dtype):
    z = randn(5, N, V, dtype=dtype)
    ids, t = teacher(6, z, 5)
    clean, cg = check(z, ids, t, temperature, tail)
    z[0, V // 2], z[1, V - 1], z[2], z[3, int(ids[3, 1])] = float("nan"), INF, -INF, float("nan")
    t[4, 2] = float("nan")
    zd, args = z.to(DEV), (ids.to(DEV), t.to(DEV))
    r = distillation_loss(zd, *args, temperature, tail)
    g = distillation_loss_backward(zd, *args, r.stats, randn(91, N).to(DEV), temperature, tail)
    loss = r.loss.cpu()
    assert bool(torch.isnan(loss[[0, 1, 3, 4]]).all()) and bool(torch.isnan(g[[0, 3, 4]]).all())
    assert bool(torch.isnan(g[1]).any()) and float(loss[2]) == INF and not bool(g[2].any())
    assert torch.equal(r.loss[5:], clean.loss[5:]) and torch.equal(g[5:], cg[5:])


@pytest.mark.parametrize("tail,temperature", TAILS)
@pytest.mark.parametrize("at", [-2.0 ** 30, -2.0 ** 20, 2.0 ** 18, 2.0 ** 30])
def test_logits_far_from_zero(at, tail, temperature):
    """Differences from the maximum are exact, wherever it lies."""
    z = (torch.round(randn(1, 5, 9001) * 64) * max(1.0, abs(at) * 2.0 ** -23)).clamp(-500, 500) + at
    t = teacher(2, (z - at).float(), 30)
    check(z, *t, temperature, tail)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("far", [5.0, 20.0, 60.0])
def test_a_small_rest_keeps_its_digits(far, dtype):
    """Listed tokens with almost all of the student's probability: the others' is summed, not left over."""
    z = randn(1, 4, 5000, dtype=dtype)
    ids, _ = teacher(2, z, 3)
    z.scatter_(1, ids, far)
    t = torch.log(torch.tensor([[0.5, 0.3, 0.1]])).repeat(4, 1)
    check(z, ids, t, 1.0, "bucket")
    check(z, ids, torch.log(torch.tensor([[0.5, 0.3, 0.2]])).repeat(4, 1), 1.0, "bucket")


def test_temperatures():
    z = randn(1, 5, 3001, scale=3.0)
    ids, t = teacher(2, z, 20)
    for temperature in (0.05, 0.7, 1.0, 13.0, 1e4):
        check(z, ids, t, temperature)
    # towards 0 the largest logit has it all
    cold = distillation_loss(z.to(DEV), ids[:, :1].to(DEV), t[:, :1].to(DEV), 1e-6).loss.cpu()
    best = z.argmax(-1) == ids[:, 0]
    assert torch.equal(cold == 0, best)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("tail,temperature", TAILS)
def test_strides_and_views(dtype, tail, temperature):
    wide = randn(1, 12, 520, dtype=dtype)
    ids, t = teacher(2, wide[:, 3:503], 9)
    r, g = check(wide[:, 3:503], ids, t, temperature, tail, z_dev=wide.to(DEV)[:, 3:503])
    zd, idd, td = wide[:, 3:503].to(DEV).contiguous(), ids.to(DEV), t.to(DEV)
    again = distillation_loss(zd.view(3, 4, 500), idd.view(3, 4, 9), td.view(3, 4, 9), temperature, tail)
    assert again.loss.shape == (3, 4) and again.stats.shape == (3, 4, 8) and torch.equal(again.loss.view(-1), r.loss)
    gl = randn(91, 12).to(DEV)
    g3 = distillation_loss_backward(zd.view(3, 4, 500), idd.view(3, 4, 9), td.view(3, 4, 9), again.stats, gl.view(3, 4), temperature, tail)
    assert torch.equal(g3.view(12, 500), g)
    both = torch.stack([idd, idd], 2), torch.stack([td, td], 2)
    assert torch.equal(distillation_loss(zd.t().contiguous().t(), both[0][:, :, 0], both[1][:, :, 1], temperature, tail).loss, r.loss)
    assert distillation_loss(zd[0], idd[0], td[0], temperature, tail).loss.shape == ()
    same = distillation_loss(zd[:1].expand(5, 500), idd[:1].expand(5, 9), td[:1].expand(5, 9), temperature, tail).loss
    assert torch.equal(same, same[:1].expand(5))
    none = distillation_loss(zd[:0], idd[:0], td[:0], temperature, tail)
    assert none.loss.shape == (0,)
    assert distillation_loss_backward(zd[:0], idd[:0], td[:0], none.stats, gl[:0], temperature, tail).shape == (0, 500)


def test_rows_past_32_bits():
    """A row that lies more than 2^32 bytes, and 2^31 elements, from the first."""
    V, N = 1 << 20, 2100
    z = torch.zeros((N, V), dtype=F16, device=DEV)
    z[-1] = randn(1, V, dtype=F16).to(DEV)
    last = z[-1:].cpu()
    ids, t = teacher(2, last, 8)
    many = ids.repeat(N, 1).to(DEV), t.repeat(N, 1).to(DEV)
    r = distillation_loss(z, *many, 1.0, "bucket")
    loss, off, g, bound = definition(last, ids, t, 1.0, "bucket")
    assert_within(r.loss[-1:], loss, off, "loss")
    got = distillation_loss_backward(z, *many, r.stats, torch.ones(N, device=DEV), 1.0, "bucket")
    assert_within(got[-1:], g, bound + ROUND[F16] * g.abs() + TINY[F16], "gradient")
    assert torch.equal(r.loss[0], r.loss[-2]) and torch.equal(got[0], got[-2])


@pytest.mark.parametrize("tail,temperature", TAILS)
def test_autograd_and_differences(tail, temperature):
    z = randn(1, 2, 3, 200)
    ids, t = (v.view(2, 3, -1).to(DEV) for v in teacher(2, z.view(6, 200), 10))
    leaf, gl = z.to(DEV).requires_grad_(), randn(3, 2, 3).to(DEV)
    r = distillation_loss(leaf, ids, t, temperature, tail)
    assert not r.stats.requires_grad
    (g,) = torch.autograd.grad(r.loss, leaf, gl)
    assert torch.equal(g, distillation_loss_backward(z.to(DEV), ids, t, r.stats, gl, temperature, tail))
    # differences of the definition in 64 bits: a step of 2^-14 leaves 2^-28 of the third derivative
    v, step = randn(4, 6, 200).double(), 2.0 ** -14
    up, down = (definition(z.view(6, 200).double() + s * step * v, ids.view(6, -1).cpu(), t.view(6, -1).cpu(), temperature, tail)[0]
                for s in (1, -1))
    diff = float(((up - down) * gl.cpu().view(6)).sum()) / (2 * step)
    gv = g.cpu().double().view(6, 200) * v
    assert abs(diff - float(gv.sum())) <= 2.0 ** -17 * float(gv.abs().sum()) + 2.0 ** -22
    with torch.no_grad():
        assert not distillation_loss(leaf, ids, t, temperature, tail).loss.requires_grad


def test_from_a_teachers_scores():
    """As it is used: token_logprobs of the teacher keeps its best tokens, the student's logits learn from them.  Against
    itself, and with its whole list, the divergence is 0 up to the log probabilities' rounding (2^-24 of |t| each)."""
    z = randn(1, 40, 64, scale=2.0).to(DEV)
    top = token_logprobs(z, torch.zeros(40, dtype=torch.int64, device=DEV), top_k=64)
    for tail in ("renormalise", "bucket"):
        r = distillation_loss(z, top.top_ids, top.top_logprobs, tail=tail)
        assert float(r.loss.abs().max()) <= 64 * 16 * U
        g = distillation_loss_backward(z, top.top_ids, top.top_logprobs, r.stats, torch.ones(40, device=DEV), tail=tail)
        assert float(g.abs().max()) <= 64 * 16 * U
    part = token_logprobs(z, torch.zeros(40, dtype=torch.int64, device=DEV), top_k=8)
    r = distillation_loss(z, part.top_ids, part.top_logprobs, tail="bucket")
    assert float(r.loss.abs().max()) <= 64 * 16 * U


def test_same_results_every_time_and_on_another_stream():
    for N, V in ((3, 100001), (600, 3001)):
        z = randn(1, N, V, dtype=BF16)
        ids, t = (v.to(DEV) for v in teacher(2, z, 50))
        z, gl = z.to(DEV), randn(3, N).to(DEV)

        def both():
            r = distillation_loss(z, ids, t, tail="bucket")
            return r.loss, r.stats, distillation_loss_backward(z, ids, t, r.stats, gl, tail="bucket")

        want = both()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = both()
        torch.cuda.current_stream().wait_stream(side)
        for w, g, o in zip(want, got, both()):
            assert torch.equal(w, g) and torch.equal(w, o)


@pytest.mark.parametrize("tail", ["renormalise", "bucket"])
@pytest.mark.parametrize("N", [1, 700])
def test_in_a_graph(N, tail):
    z = randn(1, N, 9001)
    ids, t = (v.to(DEV) for v in teacher(2, z, 20))
    z, gl = z.to(DEV), randn(3, N).to(DEV)

    def both():
        r = distillation_loss(z, ids, t, tail=tail)
        return r.loss, r.stats, distillation_loss_backward(z, ids, t, r.stats, gl, tail=tail)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for seed in range(4):
        new = randn(10 + seed, N, 9001)
        for old, v in zip((z, ids, t, gl), (new, *teacher(seed, new, 20), randn(seed, N))):
            old.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, both()):
            assert torch.equal(got, want)


def test_refusals():
    z = torch.zeros((2, 50), device=DEV)
    ids, t = torch.zeros((2, 3), dtype=torch.int64, device=DEV), torch.zeros((2, 3), device=DEV)
    good = dict(logits=z, teacher_ids=ids, teacher_logprobs=t)
    r = distillation_loss(**good)
    long = torch.zeros((2, 257), dtype=torch.int64, device=DEV)
    for error, change in (
            (RuntimeError, dict(logits=z.cpu())), (TypeError, dict(logits=z.double())), (ValueError, dict(logits=z[:, :0])),
            (ValueError, dict(teacher_ids=ids.int())), (ValueError, dict(teacher_ids=ids[:1])), (ValueError, dict(teacher_ids=ids[:, 0])),
            (ValueError, dict(teacher_ids=ids.cpu())), (ValueError, dict(teacher_ids=None)), (ValueError, dict(teacher_logprobs=t.double())),
            (ValueError, dict(teacher_logprobs=t[:, :2])), (ValueError, dict(teacher_logprobs=t.clone().requires_grad_())),
            (ValueError, dict(teacher_ids=ids[:, :0], teacher_logprobs=t[:, :0])), (ValueError, dict(teacher_ids=long, teacher_logprobs=long.float())),
            (ValueError, dict(temperature=0.0)), (ValueError, dict(temperature=-1.0)), (ValueError, dict(temperature=float("nan"))),
            (ValueError, dict(temperature=1e7)), (ValueError, dict(tail="drop")), (ValueError, dict(tail="bucket", temperature=2.0))):
        with pytest.raises(error):
            distillation_loss(**{**good, **change})
        with pytest.raises(error):
            distillation_loss_backward(**{**good, **change}, stats=r.stats, grad_loss=r.loss)
    for stats, gl in ((r.stats[:, :7], r.loss), (r.stats.double(), r.loss), (r.stats, r.loss[:1]), (r.stats, r.loss.half()), (None, r.loss),
                      (r.stats, None)):
        with pytest.raises(ValueError):
            distillation_loss_backward(**good, stats=stats, grad_loss=gl)


def test_derivatives_that_no_kernel_has_are_refused():
    from torch.autograd import forward_ad
    z = randn(1, 3, 60)
    ids, t = (v.to(DEV) for v in teacher(2, z, 5))
    z, gl = z.to(DEV), randn(3, 3).to(DEV)
    r = distillation_loss(z, ids, t)
    with forward_ad.dual_level():
        def dual(v):
            return forward_ad.make_dual(v, torch.ones_like(v))

        for call in (lambda: distillation_loss(dual(z), ids, t), lambda: distillation_loss(z, ids, dual(t)),
                     lambda: distillation_loss_backward(dual(z), ids, t, r.stats, gl),
                     lambda: distillation_loss_backward(z, ids, t, dual(r.stats), gl),
                     lambda: distillation_loss_backward(z, ids, t, r.stats, dual(gl))):
            with pytest.raises(NotImplementedError):
                call()
    leaf = z.clone().requires_grad_()
    g, = torch.autograd.grad(distillation_loss(leaf, ids, t).loss.square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    got = distillation_loss_backward(z, ids, t, r.stats, gl.clone().requires_grad_())
    assert got.requires_grad
    with pytest.raises(RuntimeError):
        got.sum().backward()


@pytest.mark.parametrize("lead", [(6,), (2, 3)])
def test_results_can_be_edited_in_place(lead):
    z = randn(1, 6, 70)
    ids, t = (v.view(*lead, 5).to(DEV) for v in teacher(2, z, 5))
    leaf = z.view(*lead, 70).to(DEV).requires_grad_()
    r = distillation_loss(leaf, ids, t)
    loss = r.loss
    loss *= 2.0
    loss.sum().backward()
    plain = distillation_loss(leaf.detach(), ids, t)
    want = distillation_loss_backward(leaf.detach(), ids, t, plain.stats, torch.full(lead, 2.0, device=DEV))
    assert torch.equal(loss.detach(), 2 * plain.loss) and torch.equal(leaf.grad, want)
    r.stats.zero_()                              # the caller's own; but the backward pass of a second one needs them
    r2 = distillation_loss(leaf, ids, t)
    r2.stats.zero_()
    with pytest.raises(RuntimeError):
        r2.loss.sum().backward()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("N,V", [(3, 40), (5, 8199), (2, 600001)])
def test_the_gradient_may_take_the_logits_place(N, V, dtype):
    """The C entry's grad_logits may be the logits: listed ones are read before they are written over, also where a
    workgroup goes over several rounds of columns."""
    from gptq_plus_mp_quant_amd import _native as nat
    z = randn(1, N, V, dtype=dtype)
    ids, t = (v.to(DEV) for v in teacher(2, z, 30))
    z, gl = z.to(DEV), randn(3, N).to(DEV)
    r = distillation_loss(z, ids, t, tail="bucket")
    want = distillation_loss_backward(z, ids, t, r.stats, gl, tail="bucket")
    nat.check("rq_distill_loss_grad", nat.load().rq_distill_loss_grad(
        z.data_ptr(), nat.DTYPE_CODES[dtype], N, V, V, ids.data_ptr(), t.data_ptr(), 30, 1.0, nat.TAILS["bucket"], r.stats.data_ptr(),
        gl.data_ptr(), z.data_ptr(), V, nat.raw_stream(z)))
    assert torch.equal(z, want)


@pytest.mark.parametrize("tail,temperature", TAILS)
@pytest.mark.parametrize("N,V", [(1, 2048), (1, 2049), (2, 8192), (511, 600), (3, 65536), (3, 65537), (2, 262145), (512, 70001)])
def test_every_way_a_row_is_cut(N, V, tail, temperature):
    """One small workgroup, one large one, several and a join; rows that end on the borders between them."""
    z = randn(N + V, N, V, dtype=BF16, scale=2.0)
    check(z, *teacher(V, z, 70), temperature, tail, grad=N * V < 1 << 20)


@pytest.mark.parametrize("tail,temperature", TAILS)
def test_a_teacher_scored_in_inference_mode(tail, temperature):
    """Its list trains a student as one from elsewhere does."""
    z, best = randn(1, 6, 500).to(DEV), randn(2, 6, 500).to(DEV)
    target = torch.zeros(6, dtype=torch.int64, device=DEV)
    with torch.inference_mode():
        scored = token_logprobs(best, target, top_k=9)
    plain = token_logprobs(best, target, top_k=9)
    grads = []
    for r in (plain, scored):
        leaf = z.clone().requires_grad_()
        distillation_loss(leaf, r.top_ids, r.top_logprobs, temperature, tail).loss.sum().backward()
        grads.append(leaf.grad)
    assert scored.top_ids.is_inference() and torch.equal(*grads) and bool(grads[0].any())
