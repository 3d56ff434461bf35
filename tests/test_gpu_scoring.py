"""token_logprobs and its gradient against the definitions in 64 bits.

Bounds: d = z - max is rounded once (2^-24 |d|), exp of it and the sums add a few units more, so a log
probability is off by at most 2^-21 (4 + |logprob|), an entropy by 2^-21 (4 + 2 log V); a gradient by
2^-19 of its terms' magnitudes (which hold exp(logprob), hence |logprob| units) and one rounding to the
logits' type."""
import math

import numpy as np
import pytest
import torch

from gptq_plus_mp_quant_amd import token_logprobs, token_logprobs_backward
from tests._packed import ROUND, TINY, assert_within
from tests._util import rng

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF = math.inf


def randn(seed, *shape, dtype=F32, scale=1.0):
    return (torch.from_numpy(rng(seed).standard_normal(shape, dtype=np.float32)) * scale).to(dtype)


def ints(seed, high, *shape):
    return torch.from_numpy(rng(seed).integers(0, high, shape))


def reference(z, t, k, ignore=-100):
    """logprob, entropy, top ids and log probabilities in float64, from the definitions."""
    z = z.double()
    N, V = z.shape
    m = z.amax(-1)
    empty = m == -INF
    d = z - torch.where(empty, 0.0, m)[:, None]
    ls = torch.where(empty, 1.0, d.exp().sum(-1)).log()
    lp = d - ls[:, None]
    p = torch.where(empty[:, None], 0.0, lp.exp())
    H = -torch.where(p == 0, 0.0, p * lp).sum(-1)
    inside = (t >= 0) & (t < V)
    mine = lp.gather(1, t.clamp(0, V - 1)[:, None])[:, 0]
    mine = torch.where(inside, mine, torch.nan)
    mine = torch.where(t == ignore, 0.0, mine)
    order = torch.where(torch.isnan(z), INF, z)
    ids = torch.sort(order + 0.0, dim=-1, descending=True, stable=True).indices[:, :k]
    return mine, H, ids, lp.gather(1, ids), lp, p, empty


def check(z, t, k=0, ignore=-100, z_dev=None):
    zd = z.to(DEV) if z_dev is None else z_dev
    r = token_logprobs(zd, t.to(DEV), top_k=k, ignore_index=ignore)
    mine, H, ids, top, _, _, _ = reference(z, t, k, ignore)
    u, V = 2.0 ** -21, z.shape[1]
    assert_within(r.logprob, mine, u * (4 + mine.abs()), "logprob")
    assert_within(r.entropy, H, torch.full_like(H, u * (4 + 2 * math.log(V))), "entropy")
    assert torch.equal(r.top_ids.cpu(), ids)
    assert_within(r.top_logprobs, top, u * (4 + top.abs()), "top_logprobs")
    return r


def check_grad(z, t, ignore=-100, entropy=True, z_dev=None):
    zd = z.to(DEV) if z_dev is None else z_dev
    N = z.shape[0]
    gl, gh = randn(91, N), randn(92, N) if entropy else None
    r = token_logprobs(zd, t.to(DEV), ignore_index=ignore)
    g = token_logprobs_backward(zd, t.to(DEV), r.stats, gl.to(DEV), None if gh is None else gh.to(DEV), ignore)
    assert g.dtype == z.dtype and g.shape == z.shape
    _, H, _, _, lp, p, empty = reference(z, t, 0, ignore)
    a = torch.where(t == ignore, 0.0, gl.double())
    b = torch.zeros(N).double() if gh is None else gh.double()
    delta = torch.zeros_like(lp).scatter_(1, t.clamp(0)[:, None], 1.0)
    finite = torch.where(p == 0, 0.0, lp)
    want = a[:, None] * (delta - p) - b[:, None] * p * (finite + H[:, None])
    want = torch.where(empty[:, None], 0.0, want)
    mag = a.abs()[:, None] * (delta + p) + b.abs()[:, None] * p * (finite.abs() + H[:, None])
    bound = 2.0 ** -19 * mag * (1 + finite.abs() / 8) + ROUND[z.dtype] * want.abs() + TINY[z.dtype] + 1e-38
    assert_within(g, want, bound, "gradient")
    return g


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("N,V,k", [(1, 1, 1), (1, 2, 2), (2, 3, 1), (3, 63, 20), (1, 64, 64), (4, 65, 64), (5, 500, 5),
                                   (1, 1000, 0), (1, 32003, 20), (7, 8191, 8), (2, 8193, 1), (300, 257, 4), (37, 32000, 20),
                                   (1, 128256, 64), (3, 100001, 20), (1100, 2000, 3),
                                   (2, 300001, 20), (512, 8200, 9)])
def test_shapes(N, V, k, dtype):
    z, t = randn(N + V, N, V, dtype=dtype, scale=3.0), ints(V, V, N)
    check(z, t, k)
    if N * V < 1 << 19:
        check_grad(z, t)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("order", ["up", "down", "equal", "late"])
@pytest.mark.parametrize("N,V", [(1, 40000), (600, 5000), (1, 270000)])
def test_orders(N, V, order, dtype):
    """Rows in rising, falling and equal order, and with all that counts at the end: the hardest for
    a running maximum and for a list of candidates kept on the way."""
    base = torch.arange(V, dtype=torch.float32) / V * 8.0 - 4.0
    row = {"up": base, "down": base.flip(0), "equal": torch.full((V,), 0.5), "late": torch.where(
        torch.arange(V) < V - 70, -30.0, base)}[order]
    z = row.to(dtype).expand(N, V).contiguous()
    check(z, ints(1, V, N), 20)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("steps", [2, 5, 40])
@pytest.mark.parametrize("N,V", [(3, 30000), (520, 4100)])
def test_many_equal_values(N, V, steps, dtype):
    """Few distinct values, so that the last places always go to the lowest of many equal indices."""
    z = torch.round(randn(steps, N, V) * steps / 4).to(dtype)
    check(z, ints(1, V, N), 33)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("N,V", [(6, 50), (6, 4099), (6, 70001)])
def test_masks(N, V, dtype):
    low = torch.finfo(dtype).min
    z = randn(V, N, V, dtype=dtype, scale=4.0)
    z[0, :] = -INF                                   # nothing left
    z[1, :] = -INF
    z[1, V - 3] = 2.0                                # one left
    z[2, ::2] = -INF
    z[3, 5:] = low
    z[4, :] = low                                    # everything at the lowest value: uniform
    t = torch.tensor([3, V - 3, 1, 2, 7, -100])
    r = check(z, t, 9)
    assert float(r.logprob[0]) == -INF and float(r.entropy[0]) == 0.0
    assert r.top_ids[0].tolist() == list(range(9)) and bool((r.top_logprobs[0] == -INF).all())
    assert float(r.logprob[1]) == 0.0 and float(r.entropy[1]) == 0.0
    g = check_grad(z, t)
    assert bool((g[0] == 0).all())
    t[2] = 0                                         # a masked target
    r = check(z, t, 9)
    assert float(r.logprob[2]) == -INF
    check_grad(z, t)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("V", [40, 5003, 70001])
def test_non_finite_rows(V, dtype):
    """NaN and +inf make their own row NaN; NaNs come first among the alternatives."""
    z = randn(V, 4, V, dtype=dtype)
    z[1, 7], z[1, V - 1], z[2, V // 2] = float("nan"), float("nan"), INF
    t = torch.tensor([1, 2, 3, 4])
    r = token_logprobs(z.to(DEV), t.to(DEV), top_k=4)
    good = check(z[[0, 3]], t[[0, 3]], 4)
    assert torch.equal(r.logprob[[0, 3]], good.logprob) and torch.equal(r.top_ids[[0, 3]], good.top_ids)
    for x in (r.logprob, r.entropy, r.top_logprobs):
        assert bool(torch.isnan(x[1:3]).all())
    assert r.top_ids[1].tolist()[:2] == [7, V - 1] and int(r.top_ids[2][0]) == V // 2
    rest = torch.sort(torch.where(torch.isnan(z[1]), -INF, z[1].float()), descending=True, stable=True).indices[:2]
    assert r.top_ids[1].tolist()[2:] == rest.tolist()
    g = token_logprobs_backward(z.to(DEV), t.to(DEV), r.stats, torch.ones(4, device=DEV), torch.ones(4, device=DEV))
    assert bool(torch.isnan(g[1:3]).all()) and bool(torch.isfinite(g[[0, 3]]).all())


def test_targets():
    z = randn(1, 5, 100)
    t = torch.tensor([-100, 99, 100, -1, 0])
    r = token_logprobs(z.to(DEV), t.to(DEV))
    assert float(r.logprob[0]) == 0.0 and bool(torch.isnan(r.logprob[2:4]).all())
    g = token_logprobs_backward(z.to(DEV), t.to(DEV), r.stats, torch.ones(5, device=DEV))
    assert bool((g[0] == 0).all()) and bool(torch.isnan(g[2:4]).all()) and bool(torch.isfinite(g[[1, 4]]).all())
    check(z, torch.tensor([3, 3, 5, 3, 0]), 2, ignore=3)
    check_grad(z, torch.tensor([3, 3, 5, 3, 0]), ignore=3, entropy=False)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_strides_and_views(dtype):
    wide = randn(2, 10, 1300, dtype=dtype)
    t = ints(3, 1111, 10)
    for cols in (slice(1, 1112), slice(0, 1111), slice(3, 1114)):
        check(wide[:, cols], t, 6, z_dev=wide.to(DEV)[:, cols])
        check_grad(wide[:, cols], t, z_dev=wide.to(DEV)[:, cols])
    z = wide[:, :1111].contiguous()
    flat = token_logprobs(z.to(DEV), t.to(DEV), top_k=3)
    r = token_logprobs(z.view(2, 5, 1111).to(DEV), t.view(2, 5).to(DEV), top_k=3)
    assert r.logprob.shape == r.entropy.shape == (2, 5) and r.top_ids.shape == r.top_logprobs.shape == (2, 5, 3)
    assert torch.equal(r.top_logprobs.view(10, 3), flat.top_logprobs) and torch.equal(r.logprob.view(10), flat.logprob)
    g = token_logprobs_backward(z.view(2, 5, 1111).to(DEV), t.view(2, 5).to(DEV), r.stats, torch.ones((2, 5), device=DEV))
    assert g.shape == (2, 5, 1111)
    one = token_logprobs(z[4].to(DEV), t[4].to(DEV), top_k=3)
    assert one.logprob.shape == () and torch.equal(one.top_ids, flat.top_ids[4])
    none = token_logprobs(z[:0].to(DEV), t[:0].to(DEV), top_k=3)
    assert none.logprob.shape == (0,) and none.top_ids.shape == (0, 3)
    check(z.t().contiguous().t(), t, 3, z_dev=z.to(DEV).t().contiguous().t())


def test_rows_past_32_bits():
    """2^31 elements and more between the first and the last row."""
    N, V, ld = 5, 1000, 600_000_000
    z = torch.empty((N - 1) * ld + V, dtype=F16, device=DEV).as_strided((N, V), (ld, 1))
    src = randn(4, N, V, dtype=F16)
    z.copy_(src)
    check(src, ints(5, V, N), 5, z_dev=z)


def test_autograd_and_differences():
    z = randn(6, 3, 4, 61, scale=2.0).to(DEV).requires_grad_()
    t = ints(7, 61, 3, 4).to(DEV)
    t[1, 2] = -100
    gl, gh = randn(8, 3, 4).to(DEV), randn(9, 3, 4).to(DEV)
    r = token_logprobs(z, t, top_k=2)
    assert not r.top_logprobs.requires_grad and not r.stats.requires_grad
    (g,) = torch.autograd.grad([r.logprob, r.entropy], z, [gl, gh])
    with torch.no_grad():
        assert torch.equal(g, token_logprobs_backward(z, t, r.stats, gl, gh))
        (g1,) = torch.autograd.grad(_lp(z, t), z)
        assert torch.equal(g1, token_logprobs_backward(z, t, r.stats, torch.ones_like(gl)))
        # central differences of the 64-bit definition, h = 1e-4: error h^2 times third derivatives (< 10)
        v = randn(10, 12, 61).double()
        zc, tc, h = z.cpu().double().view(12, 61), t.cpu().view(12), 1e-4
        f = []
        for s in (h, -h):
            mine, H, *_ = reference(zc + s * v, tc, 0)
            f.append(float((mine * gl.cpu().double().view(12)).sum() + (H * gh.cpu().double().view(12)).sum()))
        slope = (f[0] - f[1]) / (2 * h)
        got = float((g.cpu().double().view(12, 61) * v).sum())
        mag = float((g.cpu().double().view(12, 61) * v).abs().sum())
        assert abs(slope - got) <= 1e-5 * mag + 1e-5


def _lp(z, t):
    with torch.enable_grad():
        return token_logprobs(z, t).logprob.sum()


def test_same_results_every_time_and_on_another_stream():
    z, t = randn(11, 9, 50000, dtype=BF16, scale=3.0).to(DEV), ints(12, 50000, 9).to(DEV)
    a = token_logprobs(z, t, top_k=10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = token_logprobs(z, t, top_k=10)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("N", [1, 700])
def test_in_a_graph(N):
    z, t = randn(13, N, 9000, scale=3.0).to(DEV), ints(14, 9000, N).to(DEV)
    gl = randn(15, N).to(DEV)

    def step():
        r = token_logprobs(z, t, top_k=5)
        return (*r, token_logprobs_backward(z, t, r.stats, gl))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        z.copy_(randn(30 + seed, N, 9000, scale=3.0))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, step()))


def test_refusals():
    z, t = torch.zeros((3, 50), device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    for error, args in ((RuntimeError, (z.cpu(), t.cpu())), (ValueError, (z, t.cpu())), (ValueError, (z, t.int())),
                        (ValueError, (z, t[:2])), (TypeError, (z.double(), t)), (ValueError, (z, t, 51)),
                        (ValueError, (z, t, -1)), (ValueError, (z[:, :0], t))):
        with pytest.raises(error):
            token_logprobs(*args)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros((1, 100), device=DEV), t[:1], top_k=65)
    s, g = torch.zeros((3, 3), device=DEV), torch.zeros(3, device=DEV)
    for args in ((z, t, s[:2], g), (z, t, s, g[:2]), (z, t, s, g.double()), (z, t, s, g, g[:1]), (z, t, s.half(), g)):
        with pytest.raises(ValueError):
            token_logprobs_backward(*args)


@pytest.mark.parametrize("dtype,mask", [(F16, -3e4), (F16, -6e4), *((d, m) for d in (BF16, F32) for m in (
    -1e6, -2.0 ** 21, -1e8, -1e9, -1e10, -1e20, -1e30, -1.7e38))])
@pytest.mark.parametrize("N,V", [(6, 50), (6, 4099), (6, 70001), (600, 4500)])
def test_finite_masks(N, V, mask, dtype):
    """Masks by any large negative number, as attention and sampling code uses them: in part of a row, in all
    but three places of it, before and after what counts, and in the whole row."""
    z = randn(V, N, V, dtype=dtype, scale=3.0)
    z[0::6, :] = mask
    for k, c in enumerate((V // 3, V // 2, V - 2)):
        z[0::6, c] = float(k)
    z[1::6, :V // 2] = mask
    z[2::6, V // 2:] = mask
    z[3::6, :] = mask
    z[4::6][torch.from_numpy(rng(V + 1).random((z[4::6].shape[0], V)) < 0.7)] = mask
    t = torch.tensor([V // 2, V - 1, 1, 7, 3, 0]).repeat(N // 6)
    r = check(z, t, 9)
    assert bool((r.logprob[3::6] + math.log(V)).abs().max() < 1e-5) and bool((r.entropy[3::6] - math.log(V)).abs().max() < 1e-5)
    if N == 6:
        check_grad(z, t)


@pytest.mark.parametrize("at", [-2.0 ** 30, -2.0 ** 22, -2.0 ** 20, -2.0 ** 18, 2.0 ** 18, 2.0 ** 20, 2.0 ** 22, 2.0 ** 30])
@pytest.mark.parametrize("order", ["up", "down", "mixed"])
def test_logits_far_from_zero(order, at):
    """A distribution of logits that lie far from zero, a few units in their last place apart."""
    N, V = 5, 9001
    step = max(abs(at) * 2.0 ** -23, 2.0 ** -6)
    k = ints(3, 24, N, V)
    k = k if order == "mixed" else k.sort(dim=-1, descending=order == "down").values
    z = (at + step * k.double()).float()
    assert torch.equal(z.double(), at + step * k.double())
    check(z, ints(4, V, N), 5)
    check_grad(z, ints(4, V, N))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("N,V", [(5, 1), (5, 40), (5, 5003), (5, 70001), (600, 40), (515, 5003), (515, 20011)])
def test_rows_with_nothing_finite(N, V, dtype):
    """All NaN, and NaN beside nothing but -inf, are NaN in all results and in the gradient; -inf alone is a
    row with nothing left."""
    z = randn(V, N, V, dtype=dtype)
    kinds = torch.arange(N) % 5
    z[kinds == 0] = float("nan")
    z[kinds == 1] = -INF
    z[(kinds == 1).nonzero()[:, 0], V // 2] = float("nan")
    z[kinds == 2] = -INF
    z[kinds == 3] = -INF
    z[(kinds == 3).nonzero()[:, 0], V - 1] = INF
    t, k = ints(1, V, N), min(4, V)
    r = token_logprobs(z.to(DEV), t.to(DEV), top_k=k)
    g = token_logprobs_backward(z.to(DEV), t.to(DEV), r.stats, torch.ones(N, device=DEV), torch.ones(N, device=DEV))
    for kind in (0, 1, 3):
        for x in (r.logprob, r.entropy, r.top_logprobs, g):
            assert bool(torch.isnan(x[kinds == kind]).all()), kind
    assert bool((r.logprob[kinds == 2] == -INF).all()) and bool((r.entropy[kinds == 2] == 0).all())
    assert bool((r.top_logprobs[kinds == 2] == -INF).all()) and bool((g[kinds == 2] == 0).all())
    assert bool(torch.isfinite(g[kinds == 4]).all()) and bool(torch.isfinite(r.logprob[kinds == 4]).all())
    at = V // 2
    first = [at] + [i for i in range(k) if i != at]
    ids = r.top_ids.cpu()
    for kind, want in ((0, list(range(k))), (1, first[:k]), (2, list(range(k))), (3, ([V - 1] + list(range(k)))[:k])):
        assert bool((ids[kinds == kind] == torch.tensor(want)).all()), kind


@pytest.mark.parametrize("lead", [(6,), (2, 3)])
def test_results_can_be_edited_in_place(lead):
    """Masking the log probabilities in place before they are summed, with a gradient as without one."""
    z, t = randn(16, *lead, 90).to(DEV), ints(17, 90, *lead).to(DEV)
    keep = (ints(18, 2, *lead) == 1).to(DEV).float()
    want = token_logprobs(z, t, top_k=2).logprob * keep
    a, b = z.clone().requires_grad_(), z.clone().requires_grad_()
    (token_logprobs(a, t).logprob * keep).sum().backward()
    r = token_logprobs(b, t, top_k=2)
    r.logprob.mul_(keep)
    with torch.no_grad():
        r.entropy.zero_()
        r.top_logprobs.zero_()
    assert torch.equal(r.logprob.detach(), want)
    r.logprob.sum().backward()
    assert torch.equal(a.grad, b.grad)
    r = token_logprobs(z, t, top_k=2)
    r.logprob.mul_(keep)
    assert torch.equal(r.logprob, want) and bool((r.entropy > 0).all())


def test_forward_mode_is_refused():
    """A tangent, which no kernel carries on, is an error, not a result without it."""
    from torch.autograd import forward_ad
    z, t, g = randn(1, 3, 50).to(DEV), ints(2, 50, 3).to(DEV), randn(3, 3).to(DEV)
    stats = token_logprobs(z, t).stats
    with forward_ad.dual_level():
        def dual(x):
            return forward_ad.make_dual(x, torch.ones_like(x))

        for call in (lambda: token_logprobs(dual(z), t), lambda: token_logprobs_backward(dual(z), t, stats, g),
                     lambda: token_logprobs_backward(z, t, dual(stats), g), lambda: token_logprobs_backward(z, t, stats, dual(g)),
                     lambda: token_logprobs_backward(z, t, stats, g, dual(g))):
            with pytest.raises(NotImplementedError):
                call()
        token_logprobs(z, t)                                 # a level alone changes nothing


def test_gradient_of_the_gradient_call_is_refused():
    """What token_logprobs_backward returns for inputs that require grad is no constant: a gradient through it is an
    error, as it is through the gradient that autograd takes."""
    z, t, g = randn(1, 3, 50).to(DEV), ints(2, 50, 3).to(DEV), randn(3, 3).to(DEV)
    stats = token_logprobs(z, t).stats
    want = token_logprobs_backward(z, t, stats, g, g)
    for k in range(3):
        args = [z, stats, g]
        args[k] = args[k].clone().requires_grad_()
        gz = token_logprobs_backward(args[0], t, args[1], args[2], g)
        assert torch.equal(gz.detach(), want) and gz.requires_grad
        with pytest.raises(RuntimeError):
            gz.sum().backward()
        with torch.no_grad():
            assert not token_logprobs_backward(args[0], t, args[1], args[2], g).requires_grad


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("N,V,k", [(512, 33000, 20), (515, 65541, 8), (512, 140003, 5), (512, 151936, 1), (512, 256000, 64)])
def test_many_rounds_a_wave(N, V, k, dtype):
    """A row's four waves take several rounds, several to a block past 131072 columns of a 16-bit type.  The rows
    are few distinct ones over again, so that the definition in 64 bits needs only those."""
    z = randn(V, 4, V, dtype=dtype, scale=3.0)
    z[1] = torch.sort(z[1].float()).values.to(dtype)
    z[2, : V - 70] = -30.0
    z[3, ::3] = -INF
    t = ints(V, V, 4)
    few = check(z, t, k)                                     # split over workgroups
    at = (torch.arange(N) % 4).to(DEV)
    r = token_logprobs(z.to(DEV)[at], t.to(DEV)[at], top_k=k)
    assert torch.equal(r.top_ids, few.top_ids[at])
    mine, H, _, top, _, _, _ = reference(z, t, k)
    u = 2.0 ** -21
    assert_within(r.logprob, mine[at.cpu()], u * (4 + mine[at.cpu()].abs()), "logprob")
    assert_within(r.entropy, H[at.cpu()], torch.full((N,), u * (4 + 2 * math.log(V))).double(), "entropy")
    assert_within(r.top_logprobs, top[at.cpu()], u * (4 + top[at.cpu()].abs()), "top_logprobs")
