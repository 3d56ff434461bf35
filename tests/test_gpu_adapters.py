"""packed_linear_lora and its gradients against the formulas in 64 bits.

Bounds: every sum's fp32 error over the sum of its terms' magnitudes (``sum_eps``; a sum of sums has both) and one
rounding to the output's type."""
import numpy as np
import pytest
import torch

from gptq_plus_mp_quant_amd import packed_linear, packed_linear_lora, packed_linear_lora_backward
from tests._packed import ROUND, TINY, assert_within, make_entry, on, sum_eps
from tests._util import rng

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def randn(seed, *shape, dtype=F32, scale=1.0):
    return (torch.from_numpy(rng(seed).standard_normal(shape, dtype=np.float32)) * scale).to(dtype)


def case(seed, T, R, C, r, n, dtype, ids="mixed"):
    """x, grad_y, lora_a, lora_b, scaling and adapter_ids (None: one adapter), on the CPU."""
    x, gy = randn(seed, T, C, dtype=dtype), randn(seed + 1, T, R, dtype=dtype)
    a, b = randn(seed + 2, n, r, C, dtype=dtype, scale=C ** -0.5), randn(seed + 3, n, R, r, dtype=dtype, scale=0.5)
    s = torch.from_numpy(rng(seed + 4).uniform(0.5, 1.5, n).astype(np.float32))
    whose = None if ids == "one" else torch.from_numpy(rng(seed + 5).integers(-1, n, T))
    return x, gy, a, b, s, whose.sort().values if ids == "runs" else whose


def formulas(x, gy, a, b, s, whose, W, bias=None):
    """y, gx, ga, gb and the bounds of their sums, in float64, token by token."""
    T, n, r = x.shape[0], a.shape[0], a.shape[1]
    R, C = W.shape
    x, gy, a, b, s = x.double(), gy.double(), a.double(), b.double(), s.double()
    whose = torch.zeros(T, dtype=torch.int64) if whose is None else whose
    eC, eR, er, eT = sum_eps(C), sum_eps(R), sum_eps(r), sum_eps(T)
    y, dy = x @ W.t(), eC * (x.abs() @ W.abs().t())
    if bias is not None:
        y, dy = y + bias.double(), dy + 2.0 ** -22 * bias.double().abs()
    gx, dx = gy @ W, eR * (gy.abs() @ W.abs())
    ga, da, gb, db = torch.zeros_like(a), torch.zeros_like(a), torch.zeros_like(b), torch.zeros_like(b)
    for t in range(T):
        i = int(whose[t])
        if i < 0:
            continue
        if i >= n:
            y[t], gx[t] = torch.nan, torch.nan
            continue
        u, v = a[i] @ x[t], b[i].t() @ gy[t]
        mu, mv = a[i].abs() @ x[t].abs(), b[i].abs().t() @ gy[t].abs()
        y[t] += s[i] * (b[i] @ u)
        dy[t] += s[i] * (eC + er) * (b[i].abs() @ mu)
        gx[t] += s[i] * (a[i].t() @ v)
        dx[t] += s[i] * (eR + er) * (a[i].abs().t() @ mv)
        ga[i] += s[i] * torch.outer(v, x[t])
        da[i] += s[i] * (eR + eT) * torch.outer(mv, x[t].abs())
        gb[i] += s[i] * torch.outer(gy[t], u)
        db[i] += s[i] * (eC + eT) * torch.outer(gy[t].abs(), mu)
    return (y, dy), (gx, dx), (ga, da), (gb, db)


def dev(t):
    return t.to(DEV) if isinstance(t, torch.Tensor) else t


def within(got, want, dt, what):
    assert got.dtype == dt
    value, bound = want
    assert_within(got, value, bound + ROUND[dt] * value.abs() + TINY[dt], what)


def check(x, gy, a, b, s, whose, entry, W, bias=None, x_dev=None, gy_dev=None):
    dt, e = x.dtype, on(entry, DEV)
    y, gx, ga, gb = formulas(x, gy, a, b, s, whose, W, bias)
    xd, gd = dev(x) if x_dev is None else x_dev, dev(gy) if gy_dev is None else gy_dev
    got = packed_linear_lora(xd, e, dev(a), dev(b), dev(whose), dev(s), bias=dev(bias))
    within(got, y, dt, "y")
    back = packed_linear_lora_backward(gd, xd, e, dev(a), dev(b), dev(whose), dev(s))
    for one, want, what in zip(back, (gx, ga, gb), ("gx", "ga", "gb")):
        within(one, want, dt, what)
    return got, back


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T,R,C,r,n,ids", [
    (1, 1, 1, 1, 1, "one"), (1, 16, 128, 16, 1, "one"), (1, 40, 200, 5, 3, "mixed"), (3, 64, 31, 4, 2, "mixed"),
    (7, 130, 1365, 5, 3, "mixed"), (16, 33, 520, 8, 16, "mixed"), (17, 48, 384, 24, 40, "mixed"), (17, 100, 96, 17, 1, "one"),
    (33, 65, 250, 64, 5, "runs"), (64, 128, 512, 16, 64, "mixed"), (65, 31, 136, 100, 2, "runs"), (130, 20, 200, 32, 7, "mixed"),
    (2, 33, 4200, 16, 3, "mixed"), (2, 40, 5000, 16, 1, "one"), (1, 8200, 96, 7, 5, "mixed"), (2, 20, 300, 9, 2, "runs"),
    (1, 4096, 8300, 16, 2, "mixed"), (40, 24, 64, 256, 3, "mixed"), (5, 300, 4200, 16, 2, "mixed"), (600, 16, 40, 3, 2, "mixed"), (9, 8200, 130, 20, 4, "mixed")])
@pytest.mark.parametrize("nbits,groups", [(4, "128"), (5, "64"), (3, "order32")])
def test_shapes(T, R, C, r, n, ids, nbits, groups, dtype):
    entry, W = make_entry(T * 7 + R + C, R, C, nbits, groups)
    check(*case(T + R, T, R, C, r, n, dtype, ids), entry, W, bias=randn(3, R, dtype=dtype) if R % 2 == 0 else None)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("nbits", [2, 3, 4, 5, 6, 7, 8, 9])
@pytest.mark.parametrize("groups", ["channel", "32", "8", "order64"])
def test_bits_and_groups(nbits, groups, dtype):
    entry, W = make_entry(nbits, 70, 777, nbits, groups)
    check(*case(nbits, 9, 70, 777, 12, 3, dtype), entry, W)


@pytest.mark.parametrize("T", [1, 5, 20, 40, 60, 260])
def test_rows_shared_by_many_waves(T):
    """Every number of waves a workgroup and row tiles a wave, with fewer and more rank tiles than waves."""
    for R, C, r in ((8200, 64, 256), (4100, 700, 100), (40, 5000, 256), (40, 64, 33)):
        entry, W = make_entry(R, R, C, 4, "channel")
        check(*case(R + T, T, R, C, r, 3, BF16), entry, W)


def test_scaling_and_a_single_adapter():
    """A number for the scaling; adapters without the leading dimension; the same without ids as with zeros."""
    entry, W = make_entry(1, 48, 160, 4, "32")
    e = on(entry, DEV)
    x, gy, a, b, _, _ = case(2, 6, 48, 160, 8, 1, F32, "one")
    y, gx, ga, gb = formulas(x, gy, a, b, torch.tensor([0.75]), None, W)
    for ids in (None, torch.zeros(6, dtype=torch.int64, device=DEV)):
        for am, bm in ((dev(a), dev(b)), (dev(a)[0], dev(b)[0])):
            within(packed_linear_lora(dev(x), e, am, bm, ids, 0.75), y, F32, "y")
            back = packed_linear_lora_backward(dev(gy), dev(x), e, am, bm, ids, 0.75)
            assert back[1].shape == am.shape and back[2].shape == bm.shape
            for one, want in zip(back, (gx, ga, gb)):
                within(one.view(want[0].shape), want, F32, "gradient")


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_tokens_without_an_adapter(dtype):
    """They get packed_linear's result and its gradient; adapters that nobody has get zeros, whatever they hold."""
    entry, W = make_entry(4, 60, 300, 4, "128")
    e = on(entry, DEV)
    x, gy, a, b, s, _ = case(5, 20, 60, 300, 6, 4, dtype)
    whose = torch.full((20,), -1, dtype=torch.int64)
    whose[3::5] = 2
    whose[4] = -(1 << 40)
    a[0], b[1], b[3, 0, 0] = float("nan"), float("inf"), float("nan")
    s[1], s[3] = float("nan"), float("inf")
    y, (gx, ga, gb) = check(x, gy, a, b, s, whose, entry, W)
    assert bool((ga.cpu()[[0, 1, 3]] == 0).all()) and bool((gb.cpu()[[0, 1, 3]] == 0).all())
    none = torch.full((20,), -1, dtype=torch.int64, device=DEV)
    assert torch.equal(packed_linear_lora(dev(x), e, dev(a), dev(b), none, dev(s)), packed_linear(dev(x), e))
    g0, ga0, gb0 = packed_linear_lora_backward(dev(gy), dev(x), e, dev(a), dev(b), none, dev(s))
    within(g0, formulas(x, gy, a, b, s, none.cpu(), W)[1], dtype, "gx")
    assert not bool(ga0.any()) and not bool(gb0.any())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T", [6, 70])
def test_non_finite_values_stay_with_their_tokens(T, dtype):
    """An adapter with an inf or NaN, a token with one, and an id that names no adapter: theirs alone."""
    entry, W = make_entry(6, 50, 260, 5, "64")
    e = on(entry, DEV)
    x, gy, a, b, s, _ = case(7, T, 50, 260, 20, 4, dtype)
    whose = torch.arange(T) % 4
    clean = packed_linear_lora(dev(x), e, dev(a), dev(b), dev(whose), dev(s))
    cx, ca, cb = packed_linear_lora_backward(dev(gy), dev(x), e, dev(a), dev(b), dev(whose), dev(s))
    a[1, 3, 7], b[2, 5, 19] = float("nan"), float("inf")
    whose[5] = 4
    x[4, 9] = float("nan")                   # adapter 0's
    y = packed_linear_lora(dev(x), e, dev(a), dev(b), dev(whose), dev(s))
    gx, ga, gb = packed_linear_lora_backward(dev(gy), dev(x), e, dev(a), dev(b), dev(whose), dev(s))
    left = torch.arange(T) % 4 == 3
    first = (torch.arange(T) % 4 == 0) & (torch.arange(T) != 4)
    for got, want in ((y, clean), (gx, cx)):
        assert torch.equal(got.cpu()[left | first], want.cpu()[left | first])
        assert bool(torch.isnan(got.cpu()[5]).all())
    assert bool(torch.isnan(y.cpu()[4]).all()) and bool(torch.isnan(y.cpu()[1]).all())
    row = torch.zeros(50, dtype=torch.bool)
    row[5] = True                            # the inf of B's row 5 goes to that row of y
    assert bool(torch.isfinite(y.cpu()[2][~row]).all()) and not bool(torch.isfinite(y.cpu()[2][row]).any())
    assert torch.equal(ga.cpu()[3], ca.cpu()[3]) and torch.equal(gb.cpu()[3], cb.cpu()[3])
    assert bool(torch.isnan(ga.cpu()[0][:, 9]).all()) and bool(torch.isfinite(ga.cpu()[0][:, :9]).all())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T", [12, 48, 100])
def test_a_token_does_not_depend_on_its_companions(T, dtype):
    """To the bit: other adapters beside it, another place in the batch's tile, none."""
    entry, _ = make_entry(8, 100, 700, 4, "128")
    e = on(entry, DEV)
    x, gy, a, b, s, whose = (dev(t) for t in case(9, T, 100, 700, 40, 9, dtype))
    y = packed_linear_lora(x, e, a, b, whose, s)
    gx = packed_linear_lora_backward(gy, x, e, a, b, whose, s)[0]
    other = torch.roll(whose, 3)
    other[5] = whose[5]
    assert torch.equal(packed_linear_lora(x, e, a, b, other, s)[5], y[5])
    assert torch.equal(packed_linear_lora_backward(gy, x, e, a, b, other, s)[0][5], gx[5])
    back = torch.arange(T - 1, -1, -1, device=DEV)
    assert torch.equal(packed_linear_lora(x[back], e, a, b, whose[back], s), y[back])
    assert torch.equal(packed_linear_lora_backward(gy[back], x[back], e, a, b, whose[back], s)[0], gx[back])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("groups", ["128", "32", "order32"])
def test_two_tokens_with_an_adapter_each(groups, dtype):
    """What one or two tokens take (their low-rank values are made where they are used): the same adapter, two, one and
    none, one that does not exist; a NaN stays with its token."""
    entry, W = make_entry(11, 70, 1100, 4, groups)
    e = on(entry, DEV)
    x, _, a, b, s, _ = case(12, 2, 70, 1100, 13, 3, dtype)
    for ids in ((1, 1), (2, 0), (-1, 2), (0, -7), (-1, -1), (1, 3)):
        whose = torch.tensor(ids)
        y = formulas(x, torch.zeros(2, 70), a, b, s, whose, W)[0]
        got = packed_linear_lora(dev(x), e, dev(a), dev(b), dev(whose), dev(s))
        within(got, y, dtype, "y")
        assert torch.equal(got[1:], packed_linear_lora(dev(x).flip(0), e, dev(a), dev(b), dev(whose).flip(0), dev(s))[:1]) or ids[1] == 3
    a[2, 4, 1099] = float("nan")
    y = packed_linear_lora(dev(x), e, dev(a), dev(b), torch.tensor([2, 0], device=DEV), dev(s))
    assert bool(torch.isnan(y[0]).all()) and bool(torch.isfinite(y[1]).all())


@pytest.mark.parametrize("T", [1, 2, 3, 20])
@pytest.mark.parametrize("size,C", [(8, 8056), (8, 8064), (8, 8184), (8, 8192), (8, 8400)])
def test_as_many_groups_as_are_staged(size, C, T):
    """Along an order, on both sides of the number of groups whose scales lie in LDS beside the low-rank values."""
    entry, W = make_entry(C, 24, C, 4, f"order{size}")
    x, gy, a, b, s, whose = case(T, T, 24, C, 16, 2, BF16)
    y = formulas(x, gy, a, b, s, whose, W)[0]
    within(packed_linear_lora(dev(x), on(entry, DEV), dev(a), dev(b), dev(whose), dev(s)), y, BF16, "y")


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_strides_and_views(dtype):
    R, C, r, n = 50, 260, 12, 3
    entry, W = make_entry(9, R, C, 5, "channel")
    e = on(entry, DEV)
    x, gy, a, b, s, whose = case(1, 12, R, C, r, n, dtype)
    want, back = check(x, gy, a, b, s, whose, entry, W)
    wide, high = torch.zeros((12, C + 9), dtype=dtype, device=DEV), torch.zeros((12, R + 3), dtype=dtype, device=DEV)
    wide[:, 1:C + 1], high[:, 3:] = dev(x), dev(gy)
    am = dev(a).transpose(1, 2).contiguous().transpose(1, 2)
    bm = torch.zeros((n, R, r + 1), dtype=dtype, device=DEV)
    bm[:, :, 1:] = dev(b)
    ids = torch.full((12, 2), 99, dtype=torch.int64, device=DEV)
    ids[:, 1] = dev(whose)
    args = e, am, bm[:, :, 1:], ids[:, 1], torch.stack([dev(s), dev(s)], 1)[:, 1]
    assert torch.equal(packed_linear_lora(wide[:, 1:C + 1], *args), want)
    for got, ref in zip(packed_linear_lora_backward(high[:, 3:], wide[:, 1:C + 1], *args), back):
        assert torch.equal(got, ref)
    assert torch.equal(packed_linear_lora(dev(x).t().contiguous().t(), *args), want)
    # one row of x for all tokens: a gradient's broadcast input
    same = dev(x)[3:4].expand(12, C)
    assert torch.equal(packed_linear_lora(same, *args), packed_linear_lora(same.contiguous(), *args))
    # leading dimensions, none, and no tokens
    y3 = packed_linear_lora(dev(x).view(2, 6, C), e, dev(a), dev(b), dev(whose).view(2, 6), dev(s))
    assert y3.shape == (2, 6, R) and torch.equal(y3.view(12, R), want)
    assert packed_linear_lora(dev(x)[0], e, dev(a), dev(b), dev(whose)[0], dev(s)).shape == (R,)
    none = packed_linear_lora_backward(dev(gy)[:0], dev(x)[:0], e, dev(a), dev(b), dev(whose)[:0], dev(s))
    assert none[0].shape == (0, C) and not bool(none[1].any()) and not bool(none[2].any())
    assert packed_linear_lora(dev(x)[:0], e, dev(a), dev(b), dev(whose)[:0], dev(s)).shape == (0, R)


@pytest.mark.parametrize("groups", ["channel", "32", "order32"])
def test_autograd_and_differences(groups):
    entry, _ = make_entry(3, 24, 96, 4, groups)
    e = on(entry, DEV)
    x, gy, a, b, s, whose = (dev(t) for t in case(1, 10, 24, 96, 7, 3, F32))
    x, gy, whose = x.view(2, 5, 96), gy.view(2, 5, 24), whose.view(2, 5)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    y = packed_linear_lora(leaves[0], e, leaves[1], leaves[2], whose, s)
    grads = torch.autograd.grad(y, leaves, gy)
    for got, want in zip(grads, packed_linear_lora_backward(gy, x, e, a, b, whose, s)):
        assert torch.equal(got, want) and got.shape == want.shape
    # y is linear in each of the three: a difference along v of any length gives <gradient, v> up to the sums' rounding,
    # at most 2^-15 of what the values' magnitudes make
    for k, (t, g) in enumerate(zip((x, a, b), grads)):
        v = randn(20 + k, *t.shape).to(DEV)
        moved = [[u + sign * v if j == k else u for j, u in enumerate((x, a, b))] for sign in (1.0, -1.0)]
        up, down = (packed_linear_lora(m[0], e, m[1], m[2], whose, s).double() for m in moved)
        diff, size = ((up - down) * gy).sum() / 2, ((up.abs() + down.abs()) * gy.abs()).sum()
        assert abs(float(diff - (g.double() * v).sum())) <= 2.0 ** -15 * float(size)
    with torch.no_grad():
        assert not packed_linear_lora(leaves[0], e, leaves[1], leaves[2], whose, s).requires_grad
    # each alone, as a training step asks for them
    for k in range(3):
        t = [leaf if j == k else leaf.detach() for j, leaf in enumerate(leaves)]
        y = packed_linear_lora(t[0], e, t[1], t[2], whose, s)
        assert torch.equal(torch.autograd.grad(y, t[k], gy)[0], grads[k])


def test_an_adapter_that_is_shared():
    """One leaf in two layers gets both gradients; accumulating over two passes adds up."""
    entry, _ = make_entry(3, 64, 64, 4, "32")
    e = on(entry, DEV)
    x, gy, a, b, _, _ = (dev(t) for t in case(1, 5, 64, 64, 4, 1, F32, "one"))
    a, b = a.requires_grad_(), b.requires_grad_()
    h = packed_linear_lora(x, e, a, b)
    packed_linear_lora(h, e, a, b).backward(gy)
    g2x, g2a, g2b = packed_linear_lora_backward(gy, h.detach(), e, a.detach(), b.detach())
    _, g1a, g1b = packed_linear_lora_backward(g2x, x, e, a.detach(), b.detach())
    assert torch.allclose(a.grad, g1a + g2a, rtol=2.0 ** -20, atol=0) and torch.allclose(b.grad, g1b + g2b, rtol=2.0 ** -20, atol=0)


def test_same_results_every_time_and_on_another_stream():
    entry, _ = make_entry(8, 300, 1500, 4, "128")
    e = on(entry, DEV)
    x, gy, a, b, s, whose = (dev(t) for t in case(3, 70, 300, 1500, 16, 6, BF16))

    def both():
        return (packed_linear_lora(x, e, a, b, whose, s), *packed_linear_lora_backward(gy, x, e, a, b, whose, s))

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    again = both()
    for w, g, o in zip(want, got, again):
        assert torch.equal(w, g) and torch.equal(w, o)


def test_in_a_graph():
    """A captured step replayed with other tokens and other adapters for them."""
    entry, _ = make_entry(8, 96, 512, 5, "channel")
    e = on(entry, DEV)
    x, gy, a, b, s, whose = (dev(t) for t in case(3, 20, 96, 512, 9, 5, F16))

    def both():
        return (packed_linear_lora(x, e, a, b, whose, s), *packed_linear_lora_backward(gy, x, e, a, b, whose, s))

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for seed in range(4):
        new = case(30 + 10 * seed, 20, 96, 512, 9, 5, F16)
        for t, v in zip((x, gy, a, b, s, whose), new):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, both()):
            assert torch.equal(got, want)


def test_refusals():
    entry, _ = make_entry(1, 16, 64, 4, "32")
    e = on(entry, DEV)
    x, gy, a, b, s, whose = (dev(t) for t in case(1, 2, 16, 64, 4, 3, F16))
    good = dict(x=x, entry=e, lora_a=a, lora_b=b, adapter_ids=whose, scaling=s)
    packed_linear_lora(**good)
    wide = torch.zeros((3, 257, 64), dtype=F16, device=DEV), torch.zeros((3, 16, 257), dtype=F16, device=DEV)
    for error, change in (
            (RuntimeError, dict(x=x.cpu())), (ValueError, dict(x=x[:, :63])), (TypeError, dict(x=x.double())),
            (ValueError, dict(lora_a=a.float())), (ValueError, dict(lora_a=a.cpu())), (ValueError, dict(lora_b=None)),
            (ValueError, dict(lora_a=a[:, :, :63])), (ValueError, dict(lora_a=a[:2])), (ValueError, dict(lora_a=a[:, :3])),
            (ValueError, dict(lora_b=b[:, :15])), (ValueError, dict(lora_a=a[0])), (ValueError, dict(lora_a=a[0, 0], lora_b=b[0, 0])),
            (ValueError, dict(lora_a=wide[0], lora_b=wide[1])), (ValueError, dict(lora_a=a[:0], lora_b=b[:0])),
            (ValueError, dict(adapter_ids=None)), (ValueError, dict(adapter_ids=whose.int())), (ValueError, dict(adapter_ids=whose[:1])),
            (ValueError, dict(adapter_ids=whose.cpu())), (ValueError, dict(adapter_ids=[0, 0])), (ValueError, dict(scaling=s[:2])),
            (ValueError, dict(scaling=s.half())), (ValueError, dict(scaling=s.cpu())), (ValueError, dict(scaling=s.clone().requires_grad_())),
            (ValueError, dict(bias=torch.zeros(15, dtype=F16, device=DEV))), (ValueError, dict(bias=torch.zeros(16, device=DEV))),
            (ValueError, dict(bias=torch.zeros(16, dtype=F16, device=DEV, requires_grad=True))),
            (ValueError, dict(entry={**e, "groupsize": 16})), (NotImplementedError, dict(entry={**e, "nbits": 10}))):
        with pytest.raises(error):
            packed_linear_lora(**{**good, **change})
        if "bias" not in change:
            with pytest.raises(error):
                packed_linear_lora_backward(gy, **{**good, **change})
    for g in (gy[:, :15], gy[:1], gy.float()):
        with pytest.raises(ValueError):
            packed_linear_lora_backward(g, **good)


def test_derivatives_that_no_kernel_has_are_refused():
    """Forward-mode tangents, a gradient of the gradients, by autograd and from the call."""
    from torch.autograd import forward_ad
    entry, _ = make_entry(3, 32, 64, 4, "32")
    e = on(entry, DEV)
    x, gy, a, b, s, whose = (dev(t) for t in case(1, 2, 32, 64, 4, 3, F32))
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for args in ((dual(x), e, a, b, whose, s), (x, e, dual(a), b, whose, s), (x, e, a, dual(b), whose, s),
                     (x, e, a, b, whose, dual(s)), (x, {**e, "scales": dual(e["scales"])}, a, b, whose, s)):
            with pytest.raises(NotImplementedError):
                packed_linear_lora(*args)
            with pytest.raises(NotImplementedError):
                packed_linear_lora_backward(gy, *args)
        with pytest.raises(NotImplementedError):
            packed_linear_lora_backward(dual(gy), x, e, a, b, whose, s)
    leaf = a.clone().requires_grad_()
    y = packed_linear_lora(x, e, leaf, b, whose, s)
    g, = torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    for got in packed_linear_lora_backward(gy.clone().requires_grad_(), x, e, a, b, whose, s):
        assert got.requires_grad
        with pytest.raises(RuntimeError):
            got.sum().backward(retain_graph=True)


def test_weight_is_what_forward_saw():
    """An entry whose tensors are exchanged in between does not matter, one changed in place is an error; weights and
    ids made in inference mode serve as well."""
    entry, _ = make_entry(3, 32, 64, 4, "32")
    other, _ = make_entry(5, 32, 64, 5, "64")
    e = on(entry, DEV)
    x, gy, a, b, s, whose = (dev(t) for t in case(1, 4, 32, 64, 4, 3, F32))
    leaf = a.clone().requires_grad_()
    want = packed_linear_lora_backward(gy, x, e, a, b, whose, s)[1]
    y = packed_linear_lora(x, e, leaf, b, whose, s)
    e.update(on(other, DEV))
    assert torch.equal(torch.autograd.grad(y, leaf, gy)[0], want)
    e = on(entry, DEV)
    for t in (x, b, whose, s, e["qweight"], e["scales"]):
        y = packed_linear_lora(x, e, leaf, b, whose, s)
        t.mul_(1)
        with pytest.raises(RuntimeError):
            y.backward(gy)
    with torch.inference_mode():
        inferred = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in on(entry, DEV).items()}
        si, wi = s.clone(), whose.clone()
    assert torch.equal(torch.autograd.grad(packed_linear_lora(x, inferred, leaf, b, wi, si), leaf, gy)[0], want)


@pytest.mark.parametrize("lead", [(), (5,), (2, 3)])
def test_results_can_be_edited_in_place(lead):
    entry, _ = make_entry(4, 24, 64, 4, "32")
    e, x, res = on(entry, DEV), randn(1, *lead, 64).to(DEV), randn(2, *lead, 24).to(DEV)
    a, b = randn(3, 1, 4, 64).to(DEV), randn(4, 1, 24, 4).to(DEV)
    leaf = x.clone().requires_grad_()
    y = packed_linear_lora(leaf, e, a, b)
    y += res
    y.sum().backward()
    plain = packed_linear_lora(x, e, a, b)
    plain += res
    assert torch.equal(y.detach(), plain) and y.shape == (*lead, 24) and leaf.grad.shape == x.shape


def test_more_adapters_than_a_launch_holds():
    """65535 adapters of 257 tiles are more workgroups than one launch takes (2^32 threads): those on both sides of the
    cut, the first and the last, and all others 0 whatever they hold."""
    n, R, C, used = 65535, 1, 32768, [0, 65278, 65279, 65534]
    entry, W = make_entry(3, R, C, 4, "128")
    e = on(entry, DEV)
    x, gy, a, b, s, _ = case(5, 6, R, C, 1, 4, BF16)
    whose = torch.tensor([2, 0, -1, 3, 1, 2])
    y, gx, ga, gb = formulas(x, gy, a, b, s, whose, W)
    many = torch.full((n, 1, C), float("nan"), dtype=BF16, device=DEV), torch.full((n, R, 1), float("nan"), dtype=BF16, device=DEV)
    scaling = torch.full((n,), float("nan"), device=DEV)
    for t, values in zip((*many, scaling), (a, b, s)):
        t[used] = dev(values)
    ids = torch.tensor([*used, -1])[whose].to(DEV)
    within(packed_linear_lora(dev(x), e, *many, ids, scaling), y, BF16, "y")
    got = packed_linear_lora_backward(dev(gy), dev(x), e, *many, ids, scaling)
    within(got[0], gx, BF16, "gx")
    for g, want in zip(got[1:], (ga, gb)):
        within(g[used], want, BF16, "gradient")
        g[used] = 0
        assert not bool(g.any())


def test_constants_made_in_inference_mode():
    """A frozen part's activations and half an adapter from there: the other half is trained as ever."""
    entry, _ = make_entry(3, 32, 64, 4, "32")
    e = on(entry, DEV)
    x, gy, a, b, s, whose = (dev(t) for t in case(1, 4, 32, 64, 4, 3, F32))
    want = packed_linear_lora_backward(gy, x, e, a, b, whose, s)
    with torch.inference_mode():
        xi, ai, bi = x.clone(), a.clone(), b.clone()
    for args, leaf, k in (((xi, e, a.clone().requires_grad_(), bi), 2, 1), ((xi, e, ai, b.clone().requires_grad_()), 3, 2),
                          ((x.clone().requires_grad_(), e, ai, bi), 0, 0)):
        assert torch.equal(torch.autograd.grad(packed_linear_lora(*args, whose, s), args[leaf], gy)[0], want[k])


@pytest.mark.parametrize("T", [512, 513, 1100])
def test_as_many_low_rank_products_as_ride_along(T):
    """On both sides of the number of tokens from which the gradients' low-rank products get a launch of their own beside
    dx (4096 rows of its grid), with dx in one launch of 256 tokens after the other: all three gradients, and dx alone."""
    entry, W = make_entry(T, 64, 64, 4, "32")
    x, gy, a, b, s, whose = case(T, T, 64, 64, 256, 16, BF16)
    e, back = on(entry, DEV), check(x, gy, a, b, s, whose, entry, W)[1]
    leaf = dev(x).requires_grad_()
    assert torch.equal(torch.autograd.grad(packed_linear_lora(leaf, e, dev(a), dev(b), dev(whose), dev(s)), leaf, dev(gy))[0], back[0])
