"""packed_gated and its gradient against the formulas in 64 bits.

Bounds: a sum's fp32 error over the sum of its terms' magnitudes (``sum_eps``) and one rounding to the output's type.
The activation and its derivative are off by 2^-20 (1 + a^2) of their terms' magnitudes: an exponent of up to a^2 that is
rounded to 24 bits changes its power by a^2 times as much, and a few units are the functions' own; below 2^-120 they
may be 0."""
import math

import numpy as np
import pytest
import torch

from gptq_plus_mp_quant_amd import packed_gated, packed_gated_backward, packed_linear, packed_linear_lora
from tests._packed import ROUND, TINY, assert_within, make_entry, on, sum_eps
from tests._util import rng

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
ACTS = ("silu", "gelu", "gelu_tanh")


def randn(seed, *shape, dtype=F32, scale=1.0):
    return (torch.from_numpy(rng(seed).standard_normal(shape, dtype=np.float32)) * scale).to(dtype)


def activation(name, a):
    """act(a), act'(a) and the magnitudes of the derivative's terms, in float64."""
    if name == "silu":
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s)), s * (1 + a.abs() * (1 - s))
    if name == "gelu":
        s, d = 0.5 * torch.special.erfc(-a / math.sqrt(2)), torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
        return a * s, s + a * d, s + a.abs() * d
    k = 2 * math.sqrt(2 / math.pi)
    s = torch.sigmoid(k * (a + 0.044715 * a ** 3))
    d = s * torch.sigmoid(-k * (a + 0.044715 * a ** 3)) * k * (1 + 3 * 0.044715 * a * a)
    return a * s, s + a * d, s + a.abs() * d


def act_eps(a):
    return 2.0 ** -20 * (1 + a * a)


def pair(seed, I, C, nbits=(4, 4), groups=("128", "128")):
    return [make_entry(seed + 50 * k, I, C, nb, g) for k, (nb, g) in enumerate(zip(nbits, groups))]


def finite(want, bound, got):
    """fp16 values past the type's range round to infinity (65520 lies half way to the next value that the format would
    have); as near to its end as the bound, they may."""
    if got.dtype != F16:
        return want
    past = (want.abs() - bound >= 65520.0) | ((want.abs() + bound >= 65520.0) & torch.isinf(got.cpu()))
    return torch.where(past, want.sign() * math.inf, want)


def check(x, weights, act, x_dev=None):
    dt, (_, Wg), (_, Wu) = x.dtype, *weights
    g, u = (on(e, DEV) for e, _ in weights)
    xd = x.to(DEV) if x_dev is None else x_dev
    h, pre = packed_gated(xd, g, u, act, return_pre=True)
    assert h.dtype == dt and pre.dtype == F32 and h.shape == (*x.shape[:-1], Wg.shape[0])
    assert torch.equal(packed_gated(xd, g, u, act), h)
    xd, eps = x.double(), sum_eps(Wg.shape[1])
    a, b = xd @ Wg.t(), xd @ Wu.t()
    da, db = eps * (xd.abs() @ Wg.abs().t()), eps * (xd.abs() @ Wu.abs().t())
    assert_within(pre, torch.stack([a, b], -2), torch.stack([da, db], -2) + 1e-38, "pre")
    f, _, _ = activation(act, a)
    # |act'| <= 1.13
    bound = 1.13 * da * (b.abs() + db) + f.abs() * (db + act_eps(a) * b.abs()) + 2.0 ** -120 * b.abs()
    want = finite(f * b, bound, h)
    assert_within(h, want, bound + ROUND[dt] * (f * b).abs() + TINY[dt] + 1e-38, "h")
    return h, pre


def check_grad(gh, pre, weights, act, gh_dev=None):
    dt, (_, Wg), (_, Wu) = gh.dtype, *weights
    gd = gh.to(DEV) if gh_dev is None else gh_dev
    gx = packed_gated_backward(gd, pre.to(DEV), *(on(e, DEV) for e, _ in weights), act)
    assert gx.dtype == dt
    g, a, b = gh.double(), pre.double()[..., 0, :], pre.double()[..., 1, :]
    f, df, mdf = activation(act, a)
    low = 2.0 ** -120 * g.abs() * (1 + b.abs())
    want = (g * b * df) @ Wg + (g * f) @ Wu
    bound = (act_eps(a) * (g * b).abs() * mdf + low) @ Wg.abs() + (act_eps(a) * (g * f).abs() + low) @ Wu.abs()
    bound += sum_eps(2 * Wg.shape[0]) * ((g * b * df).abs() @ Wg.abs() + (g * f).abs() @ Wu.abs())
    assert_within(gx, finite(want, bound, gx), bound + ROUND[dt] * want.abs() + TINY[dt] + 1e-38, "gx")
    return gx


def pre_of(seed, T, I, scale=2.0):
    return randn(seed, T, 2, I, scale=scale)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T,I,C", [(1, 1, 1), (1, 16, 128), (1, 17, 129), (2, 3, 7), (5, 33, 520), (7, 130, 1365), (16, 15, 256),
                                   (17, 48, 384), (33, 65, 250), (64, 128, 512), (65, 31, 136), (130, 20, 200), (3, 600, 100)])
@pytest.mark.parametrize("nbits,groups", [(4, "channel"), (4, "128"), (5, "64"), (3, "order32")])
def test_shapes(T, I, C, nbits, groups, dtype):
    act, weights = ACTS[(T + I + nbits) % 3], pair(T * 7 + I + C, I, C, (nbits,) * 2, (groups,) * 2)
    check(randn(T + C, T, C, dtype=dtype), weights, act)
    check_grad(randn(T + I, T, I, dtype=dtype), pre_of(T, T, I), weights, act)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("nbits,groups", [((2, 2), ("channel", "32")), ((4, 5), ("128", "128")), ((3, 8), ("order64", "channel")),
                                          ((6, 6), ("order8", "order64")), ((7, 7), ("100", "8")), ((9, 9), ("256", "channel")),
                                          ((8, 8), ("128", "256")), ((4, 4), ("32", "64")), ((5, 2), ("channel", "order100"))])
def test_each_weight_has_its_own_bits_and_groups(nbits, groups, dtype):
    """Of one kind (one launch) and of two (one after the other)."""
    weights = pair(1, 70, 777, nbits, groups)
    for T in (3, 40):
        check(randn(T, T, 777, dtype=dtype), weights, "silu")
        check_grad(randn(T + 1, T, 70, dtype=dtype), pre_of(2, T, 70), weights, "gelu")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_the_whole_range_of_the_activation(act, dtype):
    """Projections from -200 to 200 and next to 0: the tails, where the value is a small power, and the bend."""
    I, C = 64, 128
    entry, W = make_entry(3, I, C, 4, "channel")
    x = torch.zeros((1, C), dtype=dtype)
    x[0, :2] = torch.tensor([1.0, 0.5])
    weights = []
    for k in range(2):
        from oracle.packing import pack_rows
        codes = np.zeros((I, C), dtype=np.int64)
        codes[:, 0], codes[:, 1] = np.arange(I) % 15 - 7, np.arange(I) // 8 - 4
        scales = torch.tensor([[4.0 ** (i % 5 - 2) if k == 0 else 1.0 for i in range(I)]])
        e = dict(entry, qweight=torch.from_numpy(pack_rows(codes, 4).view(np.int32)), scales=scales)
        weights.append((e, torch.from_numpy(codes) * scales.double().t()))
    _, pre = check(x, weights, act)
    check_grad(randn(5, 1, I, dtype=dtype), pre.cpu(), weights, act)
    a = torch.cat([torch.linspace(-30, 30, 500), torch.tensor([-200.0, -100.0, -88.8, -14.2, -13.1, 100.0, 200.0, 0.0, -0.0, 1e-30])])
    I = a.numel()
    pre = torch.stack([a, torch.ones(I)])[None]
    e, _ = make_entry(4, I, I, 4, "channel")
    codes = np.eye(I, dtype=np.int64)
    one = dict(e, qweight=torch.from_numpy(pack_rows(codes, 4).view(np.int32)), scales=torch.ones(1, I))
    zero = dict(one, qweight=torch.from_numpy(pack_rows(0 * codes, 4).view(np.int32)))
    for gate, up in ((one, zero), (zero, one)):              # the derivative, then the value, each by itself
        weights = [(w, torch.from_numpy(codes).double() if w is one else torch.zeros(I, I).double()) for w in (gate, up)]
        check_grad(torch.ones((1, I), dtype=dtype), pre, weights, act)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T", [1, 12, 30, 50])
@pytest.mark.parametrize("I,C,nbits,groups", [(33, 17000, 4, "128"), (40, 8400, 5, "channel"), (20, 8232, 4, "8"), (24, 8400, 4, "order8")])
def test_many_chunks_a_wave(I, C, nbits, groups, T, dtype):
    weights = pair(I, I, C, (nbits,) * 2, (groups,) * 2)
    check(randn(T, T, C, dtype=dtype, scale=0.1), weights, "silu")


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T", [3, 20, 60, 100])
def test_gradient_many_steps(T, dtype):
    """Steps of 32 rows past a wave's share, and parts past the first."""
    weights = pair(T, 9000, 130, (4, 4), ("channel", "channel"))
    check_grad(randn(T, T, 9000, dtype=dtype), pre_of(T, T, 9000), weights, "silu")


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T", [3, 17, 32, 48, 50])
@pytest.mark.parametrize("nbits", [4, 7])
def test_many_rows(nbits, T, dtype):
    """Two row tiles of each weight a wave, the last of them moved back; every number of token tiles."""
    weights = pair(T, 16408, 200, (nbits,) * 2, ("channel", "channel"))
    check(randn(T, T, 200, dtype=dtype), weights, "silu")


@pytest.mark.parametrize("groups", [("128", "128"), ("32", "order32")])
@pytest.mark.parametrize("T", [256, 257, 300, 600])
def test_more_tokens_than_a_launch(T, groups):
    dtype = (F16, BF16, F32)[T % 3]
    weights = pair(T, 40, 300, (4, 4), groups)
    check(randn(T, T, 300, dtype=dtype), weights, "gelu")
    check_grad(randn(T + 1, T, 40, dtype=dtype), pre_of(T, T, 40), weights, "gelu")


@pytest.mark.parametrize("groups", ["128", "32", "order32"])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_non_finite_inputs_stay_in_their_row(dtype, groups):
    weights = pair(21, 40, 300, (3, 3), (groups,) * 2)
    g, u = (on(e, DEV) for e, _ in weights)
    x = randn(1, 5, 300, dtype=dtype)
    clean = packed_gated(x.to(DEV), g, u)
    x[1, 7], x[3, 299] = float("inf"), float("nan")
    h = packed_gated(x.to(DEV), g, u).cpu()
    keep = [0, 2, 4]
    assert torch.equal(h[keep], clean.cpu()[keep]) and not bool(torch.isfinite(h[1]).all()) and bool(torch.isnan(h[3]).all())
    gh, pre = randn(2, 5, 40, dtype=dtype).to(DEV), pre_of(3, 5, 40).to(DEV)
    clean = packed_gated_backward(gh, pre, g, u)
    gh[1, 3], pre[3, 0, 39] = float("inf"), float("nan")
    gx = packed_gated_backward(gh, pre, g, u)
    assert torch.equal(gx[keep], clean[keep]) and bool(torch.isnan(gx[3]).all()) and not bool(torch.isfinite(gx[1]).any())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_strides_and_views(dtype):
    I, C = 50, 260
    weights = pair(9, I, C, (5, 5), ("channel", "channel"))
    g, u = (on(e, DEV) for e, _ in weights)
    wide = randn(1, 12, C + 9, dtype=dtype)
    for x in (wide[:, 1:C + 1], wide[::2, 5:C + 5], wide[3:4, :C].expand(4, C)):
        check(x, weights, "silu", x_dev=torch.as_strided(wide.to(DEV), x.shape, x.stride(), x.storage_offset()))
    gh, pre = randn(2, 12, I + 3, dtype=dtype), pre_of(3, 12, I)
    gx = check_grad(gh[:, 3:], pre, weights, "gelu", gh_dev=gh.to(DEV)[:, 3:])
    swapped = pre.to(DEV).flip(1).contiguous().flip(1).transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(packed_gated_backward(gh.to(DEV)[:, 3:], swapped, g, u, "gelu"), gx)
    x3 = wide[:6, :C].to(DEV)
    h, pre3 = packed_gated(x3.view(2, 3, C), g, u, return_pre=True)
    assert h.shape == (2, 3, I) and pre3.shape == (2, 3, 2, I)
    assert torch.equal(h.view(6, I), packed_gated(x3, g, u))
    gh3 = gh[:6, :I].to(DEV).contiguous()
    gx3 = packed_gated_backward(gh3.view(2, 3, I), pre3, g, u)
    assert gx3.shape == (2, 3, C) and torch.equal(gx3.view(6, C), packed_gated_backward(gh3, pre3.view(6, 2, I), g, u))
    assert packed_gated(x3[0], g, u).shape == (I,)
    h0, pre0 = packed_gated(x3[:0], g, u, return_pre=True)
    assert h0.shape == (0, I) and pre0.shape == (0, 2, I)
    assert packed_gated_backward(h0, pre0, g, u).shape == (0, C)
    longer = torch.full((I, g["qweight"].shape[1] + 3), -1, dtype=torch.int32, device=DEV)
    longer[:, 1:-2] = g["qweight"]
    assert torch.equal(packed_gated(x3, {**g, "qweight": longer[:, 1:-2]}, u), h.view(6, I))
    # one weight for both
    assert torch.equal(packed_gated(x3, g, {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in g.items()}),
                       packed_gated(x3, g, g))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("groups", [("32", "32"), ("channel", "order32")])
def test_autograd_and_differences(act, groups):
    weights = pair(3, 24, 96, (4, 4), groups)
    g, u = (on(e, DEV) for e, _ in weights)
    x, gh = randn(1, 2, 5, 96, scale=0.5).to(DEV).requires_grad_(), randn(2, 2, 5, 24).to(DEV)
    h = packed_gated(x, g, u, act)
    (gx,) = torch.autograd.grad(h, x, gh)
    h2, pre = packed_gated(x, g, u, act, return_pre=True)
    assert torch.equal(h, h2) and not pre.requires_grad
    assert torch.equal(gx, packed_gated_backward(gh, pre, g, u, act))
    # against differences of the formula in 64 bits along a direction: a step of 2^-14 leaves 2^-28 of the third derivative
    v = randn(5, 10, 96).double()
    Wg, Wu = (w for _, w in weights)

    def loss(xd):
        return float((activation(act, xd @ Wg.t())[0] * (xd @ Wu.t()) * gh.cpu().double().view(10, 24)).sum())

    xd, step = x.detach().cpu().double().view(10, 96), 2.0 ** -14
    diff = (loss(xd + step * v) - loss(xd - step * v)) / (2 * step)
    size = float((gx.cpu().double().view(10, 96) * v).abs().sum())
    assert abs(diff - float((gx.cpu().double().view(10, 96) * v).sum())) <= 2.0 ** -16 * size
    with torch.no_grad():
        assert not packed_gated(x, g, u, act).requires_grad


def test_a_block_with_adapters():
    """As they are used together: the gated half, then the down projection with an adapter, and the gradients back
    through both."""
    weights = pair(3, 64, 96, (4, 4), ("32", "32"))
    down, Wd = make_entry(9, 96, 64, 4, "32")
    (g, u), d = (on(e, DEV) for e, _ in weights), on(down, DEV)
    x, res = randn(1, 5, 96, scale=0.5).to(DEV).requires_grad_(), randn(2, 5, 96).to(DEV)
    a, b = (randn(3, 1, 8, 64, scale=0.1).to(DEV).requires_grad_(), randn(4, 1, 96, 8, scale=0.1).to(DEV).requires_grad_())
    y = packed_linear_lora(packed_gated(x, g, u), d, a, b, scaling=2.0)
    y.backward(res)
    xd, ad, bd = (t.detach().cpu().double().requires_grad_() for t in (x, a[0], b[0]))
    h = torch.nn.functional.silu(xd @ weights[0][1].t()) * (xd @ weights[1][1].t())
    want = h @ Wd.t() + 2.0 * (h @ ad.t()) @ bd.t()
    want.backward(res.cpu().double())
    for got, ref in ((y, want), (x.grad, xd.grad), (a.grad[0], ad.grad), (b.grad[0], bd.grad)):
        # each sum's rounding errors are 2^-19 of its terms at most; three products in a row
        assert float((got.detach().cpu().double() - ref.detach()).norm() / ref.detach().norm()) < 2.0 ** -17


def test_same_results_every_time_and_on_another_stream():
    g, u = (on(e, DEV) for e, _ in pair(8, 300, 1500))
    x, gh = randn(1, 20, 1500, dtype=BF16).to(DEV), randn(2, 20, 300, dtype=BF16).to(DEV)
    h, pre = packed_gated(x, g, u, return_pre=True)
    gx = packed_gated_backward(gh, pre, g, u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h2, pre2 = packed_gated(x, g, u, return_pre=True)
        gx2 = packed_gated_backward(gh, pre2, g, u)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(h, h2) and torch.equal(pre, pre2) and torch.equal(gx, gx2)


@pytest.mark.parametrize("T", [6, 48])
@pytest.mark.parametrize("groups", ["128", "32", "order32"])
def test_a_token_does_not_depend_on_its_companions(groups, T):
    g, u = (on(e, DEV) for e, _ in pair(8, 100, 700, groups=(groups,) * 2))
    x, gh, pre = randn(1, T, 700, dtype=BF16).to(DEV), randn(2, T, 100, dtype=BF16).to(DEV), pre_of(3, T, 100).to(DEV)
    back = torch.arange(T - 1, -1, -1, device=DEV)
    assert torch.equal(packed_gated(x[back], g, u), packed_gated(x, g, u)[back])
    assert torch.equal(packed_gated_backward(gh[back], pre[back], g, u), packed_gated_backward(gh, pre, g, u)[back])


@pytest.mark.parametrize("groups", [("channel", "channel"), ("channel", "order64")])
def test_in_a_graph(groups):
    g, u = (on(e, DEV) for e, _ in pair(8, 96, 512, (5, 5), groups))
    x, gh = randn(1, 3, 512, dtype=F16, scale=0.1).to(DEV), randn(2, 3, 96, dtype=F16).to(DEV)

    def both():
        h, pre = packed_gated(x, g, u, return_pre=True)
        return h, pre, packed_gated_backward(gh, pre, g, u), packed_gated(x, g, u, "gelu")

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for seed in range(4):
        x.copy_(randn(10 + seed, 3, 512, dtype=F16, scale=0.1))
        gh.copy_(randn(20 + seed, 3, 96, dtype=F16))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, both()):
            assert torch.equal(got, want)


def test_two_graphs_in_turn():
    """A training step through the block and its adapter, captured twice for different numbers of tokens, the graphs
    replayed in turn and between eager steps: neither's workspaces are the other's."""
    g, u = (on(e, DEV) for e, _ in pair(8, 96, 512, (4, 4), ("128", "128")))
    d = on(make_entry(9, 64, 96, 4, "channel")[0], DEV)
    a, b = randn(3, 2, 8, 96, dtype=BF16, scale=0.1).to(DEV), randn(4, 2, 64, 8, dtype=BF16, scale=0.1).to(DEV)
    leaves = [t.requires_grad_() for t in (a, b)]

    def step(x, ids, gy):
        y = packed_linear_lora(packed_gated(x, g, u), d, *leaves, ids)
        return (y.detach(), *torch.autograd.grad(y, leaves, gy))

    def inputs(seed, T):
        return (randn(seed, T, 512, dtype=BF16, scale=0.1), torch.from_numpy(rng(seed).integers(-1, 2, T)), randn(seed + 1, T, 64, dtype=BF16))

    states, graphs, outs = [], [], []
    for T in (20, 40):
        state = [t.to(DEV) for t in inputs(T, T)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*state)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*state)
        states.append(state), graphs.append(graph), outs.append(out)
    for seed in range(3):
        for state in states:
            for t, new in zip(state, inputs(100 + 10 * seed, state[0].shape[0])):
                t.copy_(new)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for state, out in zip(states, outs):
            for got, want in zip(out, step(*state)):
                assert torch.equal(got, want)


def test_refusals():
    (e, _), (f, _) = pair(1, 16, 64, (4, 4), ("32", "32"))
    g, u = on(e, DEV), on(f, DEV)
    x, gh, pre = torch.zeros((2, 64), dtype=F16, device=DEV), torch.zeros((2, 16), dtype=F16, device=DEV), pre_of(1, 2, 16).to(DEV)
    small = on(make_entry(2, 15, 64, 4, "32")[0], DEV)
    for error, args in ((RuntimeError, (x.cpu(), g, u)), (ValueError, (x[:, :63], g, u)), (TypeError, (x.double(), g, u)),
                        (ValueError, (x, g, small)), (ValueError, (x, g, {**u, "scales": u["scales"].half()})), (RuntimeError, (x, g, f)),
                        (NotImplementedError, (x, {**g, "nbits": 10}, u)), (ValueError, (x, g, u, "relu")), (ValueError, (x, g, u, None)),
                        (ValueError, (x, {**g, "scales": g["scales"].clone().requires_grad_()}, u))):
        with pytest.raises(error):
            packed_gated(*args)
    for error, args in ((RuntimeError, (gh.cpu(), pre, g, u)), (ValueError, (gh[:, :15], pre, g, u)), (ValueError, (gh, pre.half(), g, u)),
                        (ValueError, (gh, pre[:1], g, u)), (ValueError, (gh, pre[:, :1], g, u)), (ValueError, (gh, pre.cpu(), g, u)),
                        (ValueError, (gh, None, g, u)), (ValueError, (gh, pre, g, small)), (ValueError, (gh, pre, g, u, "tanh"))):
        with pytest.raises(error):
            packed_gated_backward(*args)


def test_derivatives_that_no_kernel_has_are_refused():
    from torch.autograd import forward_ad
    g, u = (on(e, DEV) for e, _ in pair(3, 32, 64, (4, 4), ("32", "32")))
    x, gh = randn(1, 2, 64).to(DEV), randn(2, 2, 32).to(DEV)
    _, pre = packed_gated(x, g, u, return_pre=True)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: packed_gated(dual(x), g, u), lambda: packed_gated(x, {**g, "scales": dual(g["scales"])}, u),
                     lambda: packed_gated_backward(dual(gh), pre, g, u), lambda: packed_gated_backward(gh, dual(pre), g, u)):
            with pytest.raises(NotImplementedError):
                call()
    leaf = x.clone().requires_grad_()
    dx, = torch.autograd.grad(packed_gated(leaf, g, u).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    for a, b in ((gh.clone().requires_grad_(), pre), (gh, pre.clone().requires_grad_())):
        got = packed_gated_backward(a, b, g, u)
        assert got.requires_grad
        with pytest.raises(RuntimeError):
            got.sum().backward()


def test_weights_are_what_forward_saw():
    (e, _), (f, _) = pair(3, 32, 64, (4, 4), ("32", "32"))
    other = on(make_entry(5, 32, 64, 5, "64")[0], DEV)
    g, u = on(e, DEV), on(f, DEV)
    x, gh = randn(1, 2, 64).to(DEV).requires_grad_(), randn(2, 2, 32).to(DEV)
    h, pre = packed_gated(x, g, u, return_pre=True)
    want = packed_gated_backward(gh, pre, g, u)
    g.update(other)
    assert torch.equal(torch.autograd.grad(h, x, gh)[0], want)
    g = on(e, DEV)
    for t in (g["qweight"], u["scales"]):
        h = packed_gated(x, g, u)
        t.mul_(1)
        with pytest.raises(RuntimeError):
            h.backward(gh)
    with torch.inference_mode():
        inferred = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in on(e, DEV).items()}
    assert torch.equal(torch.autograd.grad(packed_gated(x, inferred, on(f, DEV)), x, gh)[0], want)


@pytest.mark.parametrize("lead", [(), (5,), (2, 3)])
def test_results_can_be_edited_in_place(lead):
    g, u = (on(e, DEV) for e, _ in pair(4, 24, 64, (4, 4), ("32", "32")))
    x, res = randn(1, *lead, 64).to(DEV), randn(2, *lead, 24).to(DEV)
    leaf = x.clone().requires_grad_()
    h = packed_gated(leaf, g, u)
    h *= res
    h.sum().backward()
    plain = packed_gated(x, g, u)
    plain *= res
    assert torch.equal(h.detach(), plain) and h.shape == (*lead, 24) and leaf.grad.shape == x.shape


def test_one_launch_agrees_with_two_products():
    """What a user wrote before: two packed linears and an activation in fp32."""
    g, u = (on(e, DEV) for e, _ in pair(6, 200, 400))
    x = randn(7, 9, 400, scale=0.3).to(DEV)
    want = torch.nn.functional.silu(packed_linear(x, g)) * packed_linear(x, u)
    got = packed_gated(x, g, u)
    assert float((got - want).norm() / want.norm()) < 2.0 ** -19
