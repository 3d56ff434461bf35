"""packed_linear, its gradient and packed_moe against the formulas in 64 bits.

Bounds: a sum's fp32 error over the sum of its terms' magnitudes (``sum_eps``), one rounding to the output's
type, and for the gradient of 16-bit tensors the weight's rounding to 16 significant bits (two bf16
pieces: 2^-16 of every term)."""
import numpy as np
import pytest
import torch

from gptq_plus_mp_quant_amd import (GPTQ, GPTQPlus, WeightQuantizer, dequantize_packed, export_packed, load_packed,
                                    packed_linear, packed_linear_backward, packed_moe, save_packed, stack_packed)
from oracle.packing import pack_rows
from tests._packed import ROUND, TINY, assert_within, make_entry, on, sum_eps
from tests._util import rng, synth

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def randn(seed, *shape, dtype=F32, scale=1.0):
    return (torch.from_numpy(rng(seed).standard_normal(shape, dtype=np.float32)) * scale).to(dtype)


def check_linear(x, entry, W, bias=None, x_dev=None):
    dt = x.dtype
    y = packed_linear(x.to(DEV) if x_dev is None else x_dev, on(entry, DEV), bias=None if bias is None else bias.to(DEV))
    assert y.dtype == dt
    xd = x.double()
    want = xd @ W.t() + (0 if bias is None else bias.double())
    mag = xd.abs() @ W.abs().t() + (0 if bias is None else bias.double().abs())
    assert_within(y, want, sum_eps(W.shape[1]) * mag + ROUND[dt] * want.abs() + TINY[dt], "y")
    return y


def check_grad(gy, entry, W, gy_dev=None):
    dt = gy.dtype
    gx = packed_linear_backward(gy.to(DEV) if gy_dev is None else gy_dev, on(entry, DEV))
    assert gx.dtype == dt
    gd = gy.double()
    want, mag = gd @ W, gd.abs() @ W.abs()
    pieces = 0.0 if dt == F32 else 2.0 ** -16
    assert_within(gx, want, (sum_eps(W.shape[0]) + pieces) * mag + ROUND[dt] * want.abs() + TINY[dt], "gx")
    return gx


SHAPES = [(1, 1, 1), (1, 16, 128), (1, 17, 129), (2, 3, 7), (3, 64, 31), (5, 33, 520), (7, 130, 1365), (8, 1, 4096),
          (15, 100, 96), (16, 15, 256), (17, 48, 384), (33, 65, 250), (64, 128, 512), (65, 31, 136), (130, 20, 200)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T,R,C", SHAPES)
@pytest.mark.parametrize("nbits,groups", [(4, "channel"), (4, "128"), (5, "64"), (3, "order32")])
def test_shapes(T, R, C, nbits, groups, dtype):
    entry, W = make_entry(T * 7 + R + C, R, C, nbits, groups)
    check_linear(randn(T + C, T, C, dtype=dtype), entry, W)
    check_grad(randn(T + R, T, R, dtype=dtype), entry, W)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("nbits", [2, 3, 4, 5, 6, 7, 8, 9])
@pytest.mark.parametrize("groups", ["channel", "32", "128", "100", "8", "256", "order64"])
def test_bits_and_groups(nbits, groups, dtype):
    R, C = 70, 777
    entry, W = make_entry(nbits, R, C, nbits, groups)
    check_linear(randn(1, 9, C, dtype=dtype), entry, W, bias=randn(2, R, dtype=dtype))
    check_grad(randn(3, 9, R, dtype=dtype), entry, W)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T", [1, 4, 40])
def test_wide(T, dtype):
    """Rows and columns past several tiles of every kernel."""
    entry, W = make_entry(11, 1040, 2304, 4, "128")
    check_linear(randn(1, T, 2304, dtype=dtype), entry, W)
    check_grad(randn(2, T, 1040, dtype=dtype), entry, W)


def test_outliers_and_scales():
    """Activations 2^12 apart and scales 2^20 apart: the sums keep fp32's precision."""
    entry, W = make_entry(5, 64, 1024, 4, "128")
    entry["scales"][::2] *= 2.0 ** -20
    W = W * torch.where(entry["g_idx"] % 2 == 0, 2.0 ** -20, 1.0).double()[None, :]
    for dt in (F16, BF16, F32):
        x = randn(3, 6, 1024)
        x[:, ::97] *= 4096.0
        check_linear(x.to(dt), entry, W)
        check_grad(randn(4, 6, 64, dtype=dt), entry, W)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_strides_and_views(dtype):
    R, C = 50, 260
    entry, W = make_entry(9, R, C, 5, "channel")
    wide = randn(1, 12, C + 9, dtype=dtype)
    for x in (wide[:, 1:C + 1], wide[::2, 5:C + 5], wide[:, :C].t().contiguous().t(), wide[3:4, :C].expand(4, C)):
        dev = wide.to(DEV)
        view = torch.as_strided(dev, x.shape, x.stride(), x.storage_offset()) if x.untyped_storage().data_ptr() == \
            wide.untyped_storage().data_ptr() else x.to(DEV)
        check_linear(x, entry, W, x_dev=view)
    g = randn(2, 12, R + 3, dtype=dtype)
    check_grad(g[:, 3:], entry, W, gy_dev=g.to(DEV)[:, 3:])
    # leading dimensions, and a packed table with longer rows
    x3 = randn(4, 2, 3, C, dtype=dtype)
    y = packed_linear(x3.to(DEV), on(entry, DEV))
    assert y.shape == (2, 3, R)
    assert torch.equal(y.view(6, R), packed_linear(x3.view(6, C).to(DEV), on(entry, DEV)))
    assert packed_linear(x3[0, 0].to(DEV), on(entry, DEV)).shape == (R,)
    e = on(entry, DEV)
    longer = torch.full((R, e["qweight"].shape[1] + 3), -1, dtype=torch.int32, device=DEV)
    longer[:, 1:-2] = e["qweight"]
    e["qweight"] = longer[:, 1:-2]
    assert torch.equal(packed_linear(x3.to(DEV), e), y)
    assert packed_linear(torch.empty((0, C), dtype=dtype, device=DEV), e).shape == (0, R)
    assert packed_linear_backward(torch.empty((0, R), dtype=dtype, device=DEV), e).shape == (0, C)


@pytest.mark.parametrize("groups", ["128", "order128"])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_non_finite_inputs_stay_in_their_row(dtype, groups):
    """An inf or NaN activation makes its own token's results what the formula gives (inf times a zero
    code is NaN) and leaves the other tokens alone."""
    entry, W = make_entry(21, 40, 300, 3, groups)
    x = randn(1, 5, 300, dtype=dtype)
    x[1, 7], x[2, 290], x[3, 299] = float("inf"), float("-inf"), float("nan")
    check_linear(x, entry, W)
    g = randn(2, 5, 40, dtype=dtype)
    g[1, 0], g[3, 39], g[4, 20] = float("-inf"), float("inf"), float("nan")
    check_grad(g, entry, W)


def test_g_idx_out_of_range_reads_as_nan():
    entry, _ = make_entry(4, 20, 64, 4, "order16")
    e = on(entry, DEV)
    e["g_idx"][5] = 4
    e["g_idx"][6] = -1
    y = packed_linear(torch.ones((2, 64), device=DEV), e)
    gx = packed_linear_backward(torch.ones((2, 20), device=DEV), e)
    assert bool(torch.isnan(y).all())
    assert torch.isnan(gx).cpu().nonzero()[:, 1].tolist() == [5, 6, 5, 6]


def test_same_results_every_time_and_on_another_stream():
    entry, _ = make_entry(8, 300, 1500, 4, "128")
    e = on(entry, DEV)
    x, g = randn(1, 20, 1500, dtype=BF16).to(DEV), randn(2, 20, 300, dtype=BF16).to(DEV)
    y, gx = packed_linear(x, e), packed_linear_backward(g, e)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2, gx2 = packed_linear(x, e), packed_linear_backward(g, e)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, y2) and torch.equal(gx, gx2)


def test_in_a_graph():
    entry, _ = make_entry(8, 96, 512, 5, "channel")
    e = on(entry, DEV)
    x, g = randn(1, 3, 512, dtype=F16).to(DEV), randn(2, 3, 96, dtype=F16).to(DEV)
    packed_linear(x, e), packed_linear_backward(g, e)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gx = packed_linear(x, e), packed_linear_backward(g, e)
    for seed in range(3):
        x.copy_(randn(10 + seed, 3, 512, dtype=F16))
        g.copy_(randn(20 + seed, 3, 96, dtype=F16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, packed_linear(x, e)) and torch.equal(gx, packed_linear_backward(g, e))


@pytest.mark.parametrize("groups", ["channel", "32", "order32"])
def test_autograd_and_differences(groups):
    entry, W = make_entry(3, 24, 96, 4, groups)
    e = on(entry, DEV)
    x = randn(1, 2, 5, 96).to(DEV).requires_grad_()
    g = randn(2, 2, 5, 24).to(DEV)
    y = packed_linear(x, e)
    (gx,) = torch.autograd.grad(y, x, g)
    assert torch.equal(gx, packed_linear_backward(g, e))
    # y is linear in x: a difference along v of any length gives <gx, v> up to the sums' rounding
    v = randn(5, 2, 5, 96).to(DEV)
    with torch.no_grad():
        diff = ((packed_linear(x + v, e) - packed_linear(x - v, e)).double() * g.double()).sum() / 2
        mag = float((x.abs().cpu().double() + v.abs().cpu().double()).view(10, 96).matmul(W.abs().t()).mul(
            g.abs().cpu().double().view(10, 24)).sum())
    assert abs(float(diff - (gx.double() * v.double()).sum())) <= 4 * sum_eps(96) * mag
    with torch.no_grad():
        assert not packed_linear(x, e).requires_grad


def _quantised(cls, R, C, bits, sym, gs, act, static, seed=5):
    X, W, s, grad = synth(seed, R, C, 2, 4, 64)
    layer = torch.nn.Linear(C, R, bias=False).to(DEV, F16)
    layer.weight.data.copy_(W.to(DEV))
    g = GPTQPlus(layer, saliency=s, gradient=grad, num_groups=2, alpha=0.0, reference_loss=0.0) if cls is GPTQPlus else \
        GPTQ(layer)
    g.quantizer = WeightQuantizer()
    g.quantizer.configure(bits, perchannel=True, sym=sym, mse=False)
    for j in range(0, 4, 2):
        g.add_batch(X[j:j + 2].to(DEV), None)
    if cls is GPTQPlus:
        g.finalize_hessian()
        g.fasterquant(blocksize=64, percdamp=0.01, groupsize=gs, actorder=act, static_groups=static)
    else:
        g.fasterquant(percdamp=0.01, groupsize=gs, actorder=act, static_groups=static)
    return g


@pytest.mark.parametrize("cls,bits,sym,gs,act,static,size", [
    (GPTQPlus, 4, False, -1, True, False, 320), (GPTQPlus, 3, True, 64, True, True, 64),
    (GPTQPlus, 4, True, 64, False, False, 64), (GPTQPlus, 4, True, 64, True, False, None),
    (GPTQ, 4, True, 64, True, True, 64), (GPTQ, 4, False, 64, True, False, None), (GPTQ, 8, False, 64, False, False, 64)])
def test_exported_entries(cls, bits, sym, gs, act, static, size, tmp_path):
    """What export_packed leaves, through a file, gives the product with the weight that
    dequantize_packed rebuilds; groupsize is there exactly where the groups are runs of columns."""
    g = _quantised(cls, 96, 320, bits, sym, gs, act, static)
    e = export_packed(g)
    assert e.get("groupsize") == size
    if size:
        assert torch.equal(e["g_idx"].cpu(), (torch.arange(320) // size).to(torch.int32))
    save_packed(str(tmp_path / "p.safetensors"), {"m": e})
    back = load_packed(str(tmp_path / "p.safetensors"), device=DEV)[0]["m"]
    assert back.get("groupsize") == size
    x = randn(7, 6, 320)
    W = dequantize_packed(back, torch.float32).cpu().double()
    y = packed_linear(x.to(DEV), back)
    want, mag = x.double() @ W.t(), x.double().abs() @ W.abs().t()
    assert_within(y, want, sum_eps(320) * mag + 2.0 ** -23 * mag, "y")
    old = {k: v for k, v in back.items() if k != "groupsize"}              # a file without the size
    assert_within(packed_linear(x.to(DEV), old), want, sum_eps(320) * mag + 2.0 ** -23 * mag, "y without groupsize")


def test_refusals():
    entry, _ = make_entry(1, 16, 64, 4, "32")
    e = on(entry, DEV)
    x = torch.zeros((2, 64), dtype=F16, device=DEV)

    def bad(error, x=x, bias=None, **change):
        with pytest.raises(error):
            packed_linear(x, {**e, **change}, bias=bias)

    bad(RuntimeError, x=x.cpu())
    bad(RuntimeError, qweight=entry["qweight"])
    bad(ValueError, x=x[:, :63])
    bad(TypeError, x=x.double())
    bad(ValueError, scales=e["scales"].half())
    bad(ValueError, scales=e["scales"][:, :15])
    bad(ValueError, qweight=e["qweight"][:, :7])
    bad(ValueError, g_idx=e["g_idx"].long())
    bad(ValueError, groupsize=16)
    bad(ValueError, groupsize=-1)
    bad(NotImplementedError, nbits=10)
    bad(NotImplementedError, nbits=1)
    bad(ValueError, bias=torch.zeros(15, dtype=F16, device=DEV))
    bad(ValueError, bias=torch.zeros(16, device=DEV))
    bad(ValueError, bias=torch.zeros(16, dtype=F16, device=DEV, requires_grad=True))
    with pytest.raises(ValueError):
        packed_linear_backward(x, e)
    with pytest.raises(ValueError):
        packed_linear(x, {**e, "qweight": e["qweight"][None], "scales": e["scales"][None], "g_idx": e["g_idx"][None]})


# --- packed_moe -------------------------------------------------------------------------------


def moe_case(seed, T, D, I, E, dtype, nbits=(4, 4, 4), groups=("128", "128", "128")):
    parts = [make_entry(seed + k, R, C, nb, gr, batch=E) for k, (R, C, nb, gr) in
             enumerate(zip((I, I, D), (D, D, I), nbits, groups))]
    router = randn(seed + 9, E, D, dtype=dtype, scale=D ** -0.5)
    return randn(seed + 8, T, D, dtype=dtype), router, parts


def check_moe(x, router, parts, K, norm):
    dt, (T, D), E = x.dtype, x.shape, router.shape[0]
    y, ids, weights = packed_moe(x.to(DEV), router.to(DEV), *(on(e, DEV) for e, _ in parts), K, norm_topk=norm,
                                 return_routing=True)
    assert y.dtype == dt and y.shape == x.shape
    xd, logits = x.double(), x.double() @ router.double().t()
    best = torch.sort(logits, dim=-1, descending=True, stable=True)
    p = torch.softmax(logits, -1).gather(1, best.indices[:, :K])
    p = p / p.sum(-1, keepdim=True) if norm else p
    got = ids.cpu().long()
    # the chosen experts, up to logits closer than their sums' rounding
    slack = sum_eps(D) * (xd.abs() @ router.double().abs().t()).amax(-1, keepdim=True)
    assert bool(((logits.gather(1, got) - best.values[:, :K]).abs() <= 2 * slack).all())
    assert all(len(set(row)) == K for row in got.tolist())
    w_tol = (4 * slack + 2.0 ** -20) * p
    assert_within(weights, p, w_tol, "weights")
    Wg, Wu, Wd = (w for _, w in parts)
    want, bound = torch.zeros((T, D), dtype=torch.float64), torch.zeros((T, D), dtype=torch.float64)
    eps, eps2 = sum_eps(D), sum_eps(I_of(parts)) + 2.0 ** -16
    for t in range(T):
        for k in range(K):
            ex = int(got[t, k])
            a, b = Wg[ex] @ xd[t], Wu[ex] @ xd[t]
            da, db = eps * (Wg[ex].abs() @ xd[t].abs()), eps * (Wu[ex].abs() @ xd[t].abs())
            silu = a * torch.sigmoid(a)
            h = silu * b
            # |silu'| <= 1.1; 2^-20 for the fp32 activation itself
            dh = 1.1 * da * (b.abs() + db) + silu.abs() * db + 2.0 ** -20 * h.abs()
            o = Wd[ex] @ h
            want[t] += p[t, k] * o
            bound[t] += p[t, k] * (Wd[ex].abs() @ (dh + eps2 * h.abs())) + w_tol[t, k] * o.abs()
    if dt == F16:  # sums past the type's range round to infinity; as near to its end as the bound, they may
        past = (want.abs() - bound >= 65520.0) | ((want.abs() + bound >= 65520.0) & torch.isinf(y.cpu()))
        want = torch.where(past, want.sign() * float("inf"), want)
    assert_within(y, want, bound + ROUND[dt] * want.abs() + TINY[dt], "y")


def I_of(parts):
    return parts[0][1].shape[1]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T,D,I,E,K", [(1, 128, 96, 4, 1), (1, 256, 128, 8, 8), (3, 130, 70, 5, 2), (7, 96, 33, 16, 4),
                                       (16, 256, 130, 3, 2), (20, 64, 64, 2, 1), (33, 128, 48, 70, 6), (70, 64, 40, 4, 3)])
@pytest.mark.parametrize("norm", [True, False])
def test_moe_shapes(T, D, I, E, K, norm, dtype):
    check_moe(*moe_case(T + D, T, D, I, E, dtype), K, norm)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("nbits,groups", [((4, 4, 4), ("channel",) * 3), ((5, 5, 5), ("128", "128", "64")),
                                          ((3, 4, 8), ("32", "channel", "order16")), ((4, 4, 4), ("order64",) * 3),
                                          ((9, 2, 6), ("channel", "128", "100")), ((8, 8, 3), ("order32", "order32", "8"))])
def test_moe_bits_and_groups(nbits, groups, dtype):
    """Mixed precision: each of the three linears may have bits and groups of its own."""
    check_moe(*moe_case(4, 6, 260, 140, 6, dtype, nbits, groups), 3, True)


def test_moe_every_token_to_one_expert():
    """All tokens choose the same experts (the others are never touched), and one token none of them."""
    x, router, parts = moe_case(6, 40, 128, 64, 9, BF16)
    x = x.abs()
    router[:] = -0.1
    router[3], router[7] = 0.5, 0.4
    x[11] = -x[11]
    check_moe(x, router, parts, 2, True)


def test_moe_ties_go_to_the_lowest_index():
    x, router, parts = moe_case(2, 5, 64, 32, 12, F16)
    router[:] = router[4]
    _, ids, weights = packed_moe(x.to(DEV), router.to(DEV), *(on(e, DEV) for e, _ in parts), 5, return_routing=True)
    assert ids.cpu().tolist() == [[0, 1, 2, 3, 4]] * 5
    assert torch.allclose(weights.cpu(), torch.full((5, 5), 0.2), atol=1e-6, rtol=0)


@pytest.mark.parametrize("K", [1, 3])
def test_moe_non_finite_token(K):
    """A NaN or inf token is NaN; the other tokens are as without it."""
    x, router, parts = moe_case(3, 6, 128, 64, 5, BF16)
    args = [on(e, DEV) for e, _ in parts]
    clean = packed_moe(x.to(DEV), router.to(DEV), *args, K)
    x[2, 5], x[4, 100] = float("nan"), float("inf")
    y, ids, _ = packed_moe(x.to(DEV), router.to(DEV), *args, K, return_routing=True)
    ids = ids.cpu()
    assert bool((ids >= 0).all()) and bool((ids < 5).all())
    assert bool(torch.isnan(y[2]).all())
    keep = [0, 1, 3, 5]
    assert torch.equal(y[keep], clean[keep])


def test_moe_views_and_stack():
    entries = [make_entry(30 + i, 48, 64, 4, "32")[0] for i in range(4)]
    gate = stack_packed([on(e, DEV) for e in entries])
    assert gate["qweight"].shape == (4, 48, 8) and gate["groupsize"] == 32
    up = stack_packed([on(make_entry(50 + i, 48, 64, 4, "32")[0], DEV) for i in range(4)])
    down = stack_packed([on(make_entry(70 + i, 64, 48, 5, "channel")[0], DEV) for i in range(4)])
    wide = randn(1, 6, 70, dtype=F16).to(DEV)
    router = randn(2, 4, 64, dtype=F16).to(DEV)
    y = packed_moe(wide[:, 3:67], router, gate, up, down, 2)
    assert torch.equal(y, packed_moe(wide[:, 3:67].contiguous(), router, gate, up, down, 2))
    y3, ids, w = packed_moe(wide[:, 3:67].contiguous().view(2, 3, 64), router, gate, up, down, 2, return_routing=True)
    assert torch.equal(y3.view(6, 64), y) and ids.shape == (2, 3, 2) and w.shape == (2, 3, 2)
    assert packed_moe(wide[:0, 3:67], router, gate, up, down, 2).shape == (0, 64)
    # one expert of one: its three packed linears in fp32
    lone = [{**e, **{k: e[k][2:3] for k in ("qweight", "scales", "g_idx")}} for e in (gate, up, down)]
    x1 = wide[:, 3:67].float().contiguous()
    first = [{k: v[0] if isinstance(v, torch.Tensor) else v for k, v in e.items()} for e in lone]
    a = packed_linear(x1, first[0])
    want = packed_linear(torch.nn.functional.silu(a) * packed_linear(x1, first[1]), first[2])
    got = packed_moe(x1, router[:1].float(), *lone, 1)
    assert float((got - want).norm() / want.norm()) < 1e-5


def test_moe_in_a_graph():
    x, router, parts = moe_case(12, 4, 128, 64, 8, F16)
    x, router, args = x.to(DEV), router.to(DEV), [on(e, DEV) for e, _ in parts]
    packed_moe(x, router, *args, 2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = packed_moe(x, router, *args, 2)
    for seed in range(3):
        x.copy_(randn(40 + seed, 4, 128, dtype=F16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, packed_moe(x, router, *args, 2))


def test_moe_refusals():
    x, router, parts = moe_case(1, 2, 64, 32, 4, F16)
    x, router = x.to(DEV), router.to(DEV)
    gate, up, down = (on(e, DEV) for e, _ in parts)
    with pytest.raises(ValueError):
        packed_moe(x, router, gate, up, down, 5)
    with pytest.raises(ValueError):
        packed_moe(x, router, gate, up, down, 0)
    with pytest.raises(ValueError):
        packed_moe(x, router.float(), gate, up, down, 2)
    with pytest.raises(ValueError):
        packed_moe(x, router[:3], gate, up, down, 2)
    with pytest.raises(ValueError):
        packed_moe(x, router, gate, up, gate, 2)
    with pytest.raises(ValueError):
        packed_moe(x, router, gate, {k: v[0] if isinstance(v, torch.Tensor) else v for k, v in up.items()}, down, 2)
    with pytest.raises(NotImplementedError):
        packed_moe(x.requires_grad_(), router, gate, up, down, 2)
    with pytest.raises(RuntimeError):
        packed_moe(x.detach().cpu(), router, gate, up, down, 2)
    with pytest.raises(ValueError):
        stack_packed([])
    with pytest.raises(ValueError):
        stack_packed([on(make_entry(1, 16, 64, 4, "32")[0], DEV), on(make_entry(1, 16, 64, 5, "32")[0], DEV)])


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("nbits", [2, 3, 4, 5, 6, 7, 8, 9])
@pytest.mark.parametrize("I", [32, 96, 140, 160])
def test_moe_widths_that_are_not_whole_chunks(I, nbits, T):
    """down's rows end inside a chunk of 128 columns (and, 140, inside a word's 32), with few and many pairs."""
    dtype = (F16, BF16, F32)[(I // 4 + nbits) % 3]
    check_moe(*moe_case(I + nbits, T, 200, I, 3, dtype, (nbits,) * 3, ("channel", "128", ("channel", "128")[nbits % 2])), 2, True)


@pytest.mark.parametrize("T,D,I,E,K", [(16, 72, 256, 5, 2), (33, 520, 384, 4, 1), (64, 130, 128, 16, 4), (100, 64, 640, 8, 3)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_moe_many_pairs(T, D, I, E, K, dtype):
    """Workgroups that share rows of down, several units an expert, more tokens than a pass takes."""
    check_moe(*moe_case(T + I, T, D, I, E, dtype, (5, 5, 4), ("128", "128", "128")), K, False)


def test_moe_most_experts():
    """As many experts and choices as there can be: the units fill most of the shared memory."""
    check_moe(*moe_case(5, 64, 32, 32, 1024, F32, (4, 4, 4), ("channel",) * 3), 64, True)


def test_moe_many_pairs_keep_to_themselves():
    """The same rows give the same bits again, and a NaN token leaves the others' as they were."""
    x, router, parts = moe_case(21, 48, 256, 384, 6, BF16)
    x, router, args = x.to(DEV), router.to(DEV), [on(e, DEV) for e, _ in parts]
    clean = packed_moe(x, router, *args, 2)
    assert torch.equal(clean, packed_moe(x, router, *args, 2))
    x[7, 3] = float("nan")
    y = packed_moe(x, router, *args, 2)
    assert bool(torch.isnan(y[7]).all())
    keep = [t for t in range(48) if t != 7]
    # the NaN token's experts have other companions now, in another order of units
    assert torch.allclose(y[keep].float(), clean[keep].float(), rtol=2.0 ** -7, atol=1e-6)


def test_second_derivatives_are_refused():
    """The gradients come from kernels that no graph follows: a gradient of them is an error, not a zero."""
    entry, _ = make_entry(3, 32, 64, 4, "32")
    x = randn(1, 2, 64).to(DEV).requires_grad_()
    g, = torch.autograd.grad(packed_linear(x, on(entry, DEV)).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("T", [1, 65])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("E,K", [(1, 1), (3, 3), (64, 5), (65, 64), (200, 7), (256, 64), (257, 6)])
def test_moe_one_token_at_a_time(E, K, norm, T):
    """A lone token (the last pass of 65 as well) at every number of experts, up to all of them chosen."""
    check_moe(*moe_case(E + K, T, 64, 48, E, (F16, BF16, F32)[E % 3], (4, 4, 4), ("32", "32", "channel")), K, norm)


def test_moe_one_token_ties_and_mixed_bits():
    x, router, parts = moe_case(7, 1, 64, 32, 100, F16, (3, 4, 5), ("32", "channel", "order16"))
    router[:] = router[4]
    router[90] = 2 * router[4] * torch.sign(router[4] @ x[0])
    _, ids, weights = packed_moe(x.to(DEV), router.to(DEV), *(on(e, DEV) for e, _ in parts), 5, return_routing=True)
    rest = [e for e in range(100) if e != 90]
    assert ids.cpu().tolist() == [[90] + rest[:4]]
    router[:, :] = 0.0
    check_moe(x, router, parts, 3, True)
    x[0, 3] = float("nan")
    y, ids, _ = packed_moe(x.to(DEV), router.to(DEV), *(on(e, DEV) for e, _ in parts), 3, return_routing=True)
    assert bool(torch.isnan(y).all()) and bool((ids >= 0).all()) and bool((ids < 100).all())


def test_single_row_with_a_short_stride():
    """One row's stride is never used: scales that are a transposed column, a weight of one row."""
    entry, W = make_entry(5, 40, 64, 4, "channel")
    e = on(entry, DEV)
    e["scales"] = e["scales"].as_strided((1, 40), (1, 1))
    check_linear(randn(1, 3, 64, dtype=F16), e, W)
    entry, W = make_entry(6, 1, 64, 4, "32")
    e = on(entry, DEV)
    e["qweight"] = e["qweight"].as_strided((1, 8), (1, 1))
    check_linear(randn(2, 3, 64, dtype=F16), e, W)
    check_grad(randn(3, 3, 1, dtype=F16), e, W)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("T", [2, 20])
def test_more_groups_than_are_staged(T, dtype):
    """Scales are read from memory where a workgroup's do not fit its share of LDS."""
    for groups, C in (("order8", 8400), ("8", 8232)):
        entry, W = make_entry(C, 24, C, 4, groups)
        check_linear(randn(T, T, C, dtype=dtype), entry, W)
        check_grad(randn(T + 1, T, 24, dtype=dtype), entry, W)


@pytest.mark.parametrize("T", [1, 24])
def test_moe_more_groups_than_are_staged(T):
    check_moe(*moe_case(T, T, 2080, 560, 3, BF16, (4, 4, 4), ("order8", "order8", "order8")), 2, True)


# --- 32 bits throughout ------------------------------------------------------------------------


def by_hand(codes, scales, g_idx, nbits, groupsize=None):
    """An entry from codes [R, C], scales [ngroups, R] and groups [C], and its weight in float64."""
    R, C = codes.shape
    entry = dict(qweight=torch.from_numpy(pack_rows(codes, nbits).view(np.int32)), scales=torch.from_numpy(scales),
                 g_idx=torch.from_numpy(g_idx.astype(np.int32)), nbits=nbits, bits=nbits, sym=True, shape=(R, C), dtype="float16")
    if groupsize:
        entry["groupsize"] = groupsize
    return entry, torch.from_numpy(scales.astype(np.float64)[g_idx].T * codes)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T", [5, 20, 40])
@pytest.mark.parametrize("nbits,groups", [(4, "channel"), (5, "128"), (4, "32"), (5, "order32")])
def test_gradient_keeps_32_bits(nbits, groups, T, dtype):
    """Two rows whose products cancel to the last bit of fp32 (codes and scales are three times as large in
    one): what is left shows every rounding to fewer bits on the way.  Allowed, in units of 2^-24 of the
    terms' magnitudes: two for the products of dy, scale and code, two for each of the sums over at most six
    pairs of pieces."""
    r, C = rng(T + nbits), 384
    size = C if groups == "channel" else int(groups.replace("order", ""))
    order = r.permutation(C) if groups.startswith("order") else np.arange(C)
    g_idx = np.argsort(order) // size
    codes = r.choice([-2, -1, 1, 2], size=(1, C))
    codes = np.concatenate([3 * codes, -codes])
    a, b = 1.375, 1.25
    s0 = (r.uniform(0.5, 1.0, size=C // size) * 0.25).astype(np.float32)
    scales = np.stack([s0, (3 * s0 * np.float32(a) / np.float32(b)).astype(np.float32)], 1)
    entry, W = by_hand(codes, scales, g_idx, nbits, None if groups.startswith("order") else size)
    gy = torch.from_numpy(r.integers(1, 16, size=(T, 1)) * np.array([[a, b]])).to(dtype)     # exact in every type
    gx = packed_linear_backward(gy.to(DEV), on(entry, DEV))
    want, mag = gy.double() @ W, gy.double().abs() @ W.abs()
    assert float((want.abs() / mag).max()) < 2.0 ** -23
    assert_within(gx, want, 14 * 2.0 ** -24 * mag + ROUND[dtype] * want.abs() + TINY[dtype], "gx")


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T", [1, 5, 40])
@pytest.mark.parametrize("I,groups", [(2, "channel"), (64, "channel"), (64, "order32"), (96, "32")])
def test_moe_activation_keeps_32_bits(I, groups, T, dtype):
    """Two columns of the activation that are one and three times the same, which down cancels: everything
    before the activation is exact (few bits, scales that are powers of two), so the result is off by the
    activation's own rounding, one unit of 2^-24, and two for each of the six pieces' products in the sum."""
    r, D, E = rng(T + I), 32, 3

    def stacked(parts):
        entry = dict(parts[0][0])
        entry.update({k: torch.stack([e[k] for e, _ in parts]) for k in ("qweight", "scales", "g_idx")})
        return entry, torch.stack([w for _, w in parts])

    def one(codes, scale, C):
        size = C if groups == "channel" else int(groups.replace("order", ""))
        g_idx = np.arange(C) // size if size < C else np.zeros(C, dtype=np.int64)
        if groups.startswith("order"):
            g_idx = g_idx[::-1].copy()
        scales = np.full((int(g_idx.max()) + 1, codes.shape[0]), scale, dtype=np.float32)
        return by_hand(codes, scales, g_idx, 4, None if groups.startswith("order") else size)

    def expert():
        gate, up, down = (np.zeros(s, dtype=np.int64) for s in ((I, D), (I, D), (D, I)))
        gate[:2] = r.integers(-7, 8, size=(1, D))
        up[:1] = r.integers(-2, 3, size=(1, D))
        up[1] = 3 * up[0]
        v = r.choice([-2, -1, 1, 2], size=D)
        down[:, 0], down[:, 1] = 3 * v, -v
        return one(gate, 2.0 ** -6, D), one(up, 2.0 ** -3, D), one(down, 2.0 ** -2, I)

    parts = [stacked(p) for p in zip(*(expert() for _ in range(E)))]
    x = torch.from_numpy(r.integers(-15, 16, size=(T, D)) / 4.0).to(dtype)
    router = randn(T, E, D, dtype=dtype)
    y, ids, w = packed_moe(x.to(DEV), router.to(DEV), *(on(e, DEV) for e, _ in parts), 1, return_routing=True)
    assert torch.equal(w.cpu(), torch.ones(T, 1))
    Wg, Wu, Wd = (p[1][ids.cpu().long()[:, 0]] for p in parts)
    xd = x.double()[:, :, None]
    gate, up = Wg @ xd, Wu @ xd
    h = gate * torch.sigmoid(gate) * up
    want, mag = (Wd @ h)[:, :, 0], (Wd.abs() @ h.abs())[:, :, 0]
    assert float(mag.max()) > 0.1 and float(want.abs().max()) <= 1e-12 * float(mag.max())
    assert_within(y, torch.zeros_like(want), 13 * 2.0 ** -24 * mag + TINY[dtype], "y")


@pytest.mark.parametrize("lead", [(), (5,), (2, 3), (2, 1, 2)])
def test_results_can_be_edited_in_place(lead):
    """A residual added in place, whatever the leading dimensions, with a gradient as without one."""
    entry, _ = make_entry(4, 24, 64, 4, "32")
    e, x, res = on(entry, DEV), randn(1, *lead, 64).to(DEV), randn(2, *lead, 24).to(DEV)
    leaf = x.clone().requires_grad_()
    y = packed_linear(leaf, e)
    y += res
    y.sum().backward()
    plain = packed_linear(x, e)
    plain += res
    assert torch.equal(y.detach(), plain) and y.shape == (*lead, 24)
    assert torch.equal(leaf.grad, packed_linear_backward(torch.ones_like(plain), e)) and leaf.grad.shape == x.shape


def test_forward_mode_is_refused():
    """A tangent, which no kernel carries on, is an error, not a result without it."""
    from torch.autograd import forward_ad
    entry, _ = make_entry(3, 32, 64, 4, "32")
    e = on(entry, DEV)
    x, g = randn(1, 2, 64).to(DEV), randn(2, 2, 32).to(DEV)
    xm, router, parts = moe_case(1, 2, 64, 32, 4, F32)
    xm, router, parts = xm.to(DEV), router.to(DEV), [on(p, DEV) for p, _ in parts]
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: packed_linear(dual(x), e), lambda: packed_linear(x, e, bias=dual(g[0])),
                     lambda: packed_linear(x, {**e, "scales": dual(e["scales"])}),
                     lambda: packed_linear_backward(dual(g), e), lambda: packed_moe(dual(xm), router, *parts, 2),
                     lambda: packed_moe(xm, dual(router), *parts, 2)):
            with pytest.raises(NotImplementedError):
                call()
        assert packed_linear(x, e).shape == (2, 32)          # a level alone changes nothing


def test_gradient_of_the_gradient_call_is_refused():
    """What packed_linear_backward returns for a grad_y that requires grad is no constant: a gradient through it is
    an error, as it is through the gradient that autograd takes."""
    entry, _ = make_entry(3, 32, 64, 4, "32")
    e, g = on(entry, DEV), randn(2, 2, 32).to(DEV)
    leaf = g.clone().requires_grad_()
    gx = packed_linear_backward(leaf, e)
    assert torch.equal(gx.detach(), packed_linear_backward(g, e)) and gx.requires_grad
    with pytest.raises(RuntimeError):
        gx.sum().backward()
    with torch.no_grad():
        assert not packed_linear_backward(leaf, e).requires_grad


def test_weight_is_what_forward_saw():
    """The gradient goes through the weight that the product was taken with: an entry whose tensors are
    exchanged in between does not matter, one changed in place is an error."""
    entry, _ = make_entry(3, 32, 64, 4, "32")
    other, _ = make_entry(5, 32, 64, 5, "64")
    e = on(entry, DEV)
    x, g = randn(1, 2, 64).to(DEV).requires_grad_(), randn(2, 2, 32).to(DEV)
    y = packed_linear(x, e)
    want = packed_linear_backward(g, e)
    e.update(on(other, DEV))
    assert torch.equal(torch.autograd.grad(y, x, g)[0], want)
    e = on(entry, DEV)
    for name in ("qweight", "scales", "g_idx"):
        y = packed_linear(x, e)
        e[name].mul_(1)
        with pytest.raises(RuntimeError):
            y.backward(g)
    with torch.inference_mode():
        e = on(entry, DEV)
        inferred = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in e.items()}
    assert torch.equal(torch.autograd.grad(packed_linear(x, inferred), x, g)[0], want)


def test_scales_that_require_grad_are_refused():
    """They would get none, as a bias would."""
    entry, _ = make_entry(3, 32, 64, 4, "32")
    e = on(entry, DEV)
    e["scales"].requires_grad_()
    x, g = randn(1, 2, 64).to(DEV), randn(2, 2, 32).to(DEV)
    xm, router, parts = moe_case(1, 2, 64, 32, 4, F32)
    xm, router, parts = xm.to(DEV), router.to(DEV), [on(p, DEV) for p, _ in parts]
    for call in (lambda: packed_linear(x, e), lambda: packed_linear(x.clone().requires_grad_(), e), lambda: packed_linear_backward(g, e)):
        with pytest.raises(ValueError):
            call()
    for k in range(3):
        changed = list(parts)
        changed[k] = {**parts[k], "scales": parts[k]["scales"].clone().requires_grad_()}
        with pytest.raises(ValueError):
            packed_moe(xm, router, *changed, 2)
        with torch.no_grad():
            assert torch.equal(packed_moe(xm, router, *changed, 2), packed_moe(xm, router, *parts, 2))
    with torch.no_grad():
        assert packed_linear(x, e).shape == (2, 32)


def test_groups_of_millions_of_columns():
    """Group sizes whose division by multiplication would not hold in 32 bits."""
    size = 32 * 100020                   # a multiple of 128; 100020^2 is past 2^32
    C = 2 * size
    r = rng(1)
    q = torch.from_numpy(r.integers(0, 1 << 32, size=(1, C // 8), dtype=np.uint32).view(np.int32))
    e = dict(qweight=q.to(DEV), scales=torch.tensor([[0.5], [2.0]], device=DEV), nbits=4,
             g_idx=(torch.arange(C, device=DEV) // size).to(torch.int32), groupsize=size)
    nibbles = torch.from_numpy(np.ascontiguousarray(q.numpy().view(np.uint8))).view(-1)
    codes = torch.stack((nibbles & 15, nibbles >> 4), 1).view(-1).double() - 8
    W = codes * torch.where(torch.arange(C) < size, 0.5, 2.0)
    gx = packed_linear_backward(torch.ones((1, 1), device=DEV), e)
    assert torch.equal(gx.cpu().double(), W[None])
    x = torch.zeros((2, C))
    x[0, ::7], x[1, size - 200:size + 200] = 1.0, 1.0
    want, mag = x.double() @ W, x.double() @ W.abs()
    assert bool(((packed_linear(x.to(DEV), e).cpu().double()[:, 0] - want).abs() <= sum_eps(C) * mag).all())


def test_strides_that_no_element_needs():
    """One word a row, or one row: the stride along it is never used, and tables that come transposed have any."""
    entry, W = make_entry(5, 20, 8, 4, "channel")
    e = on(entry, DEV)
    e["qweight"] = e["qweight"].as_strided((20, 1), (1, 20))
    check_linear(randn(1, 3, 8, dtype=F16), e, W)
    check_grad(randn(2, 3, 20, dtype=F16), e, W)
    entry, W = make_entry(6, 1, 96, 4, "32")
    e = on(entry, DEV)
    e["scales"] = e["scales"].as_strided((3, 1), (1, 3))
    check_linear(randn(3, 3, 96, dtype=F16), e, W)
    check_grad(randn(4, 3, 1, dtype=F16), e, W)
    parts = [make_entry(7 + k, R, C, 4, "channel", batch=2) for k, (R, C) in enumerate(((1, 8), (1, 8), (8, 1)))]
    x, router = randn(8, 2, 8, dtype=F16), randn(9, 2, 8, dtype=F16)
    want = packed_moe(x.to(DEV), router.to(DEV), *(on(e, DEV) for e, _ in parts), 1)
    odd = [on(e, DEV) for e, _ in parts]
    odd[0]["qweight"] = odd[0]["qweight"].as_strided((2, 1, 1), (1, 1, 5))
    odd[1]["scales"] = odd[1]["scales"].as_strided((2, 1, 1), (1, 1, 7))
    odd[2]["qweight"] = odd[2]["qweight"].as_strided((2, 8, 1), (8, 1, 3))
    assert torch.equal(packed_moe(x.to(DEV), router.to(DEV), *odd, 1), want)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T", [1, 12, 30, 50])
@pytest.mark.parametrize("R,C,nbits,groups,times", [(48, 17000, 4, "128", 1), (33, 17160, 5, "channel", 1), (41, 8400, 4, "128", 200)])
def test_many_chunks_a_wave(R, C, nbits, groups, times, T, dtype):
    """Waves that take eight chunks of 128 columns and more, so that the loop that refills what is in flight
    runs; with one row tile a wave and (R * times >= 8192) with two."""
    entry, W = make_entry(R + nbits, R, C, nbits, groups)
    x = randn(T, T, C, dtype=dtype)
    y = check_linear(x, entry, W)
    if times > 1:
        e = on(entry, DEV)
        e["qweight"], e["scales"] = e["qweight"].repeat(times, 1), e["scales"].repeat(1, times)
        many = packed_linear(x.to(DEV), e).view(T, times, R)
        assert torch.equal(many, many[:, :1].expand_as(many))
        xd = x.double()
        want, mag = xd @ W.t(), xd.abs() @ W.abs().t()
        assert_within(many[:, 0], want, sum_eps(C) * mag + ROUND[dtype] * want.abs() + TINY[dtype], "y")
    assert y.shape == (T, R)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T", [9, 60])
def test_gradient_many_steps(T, dtype):
    """Waves that take seven steps of 32 rows and more: 14336 columns, the same 128 over again."""
    R, times = 9000, 112
    entry, W = make_entry(T, R, 128, 4, "channel")
    g = randn(T, T, R, dtype=dtype)
    e = on(entry, DEV)
    e["qweight"], e["g_idx"], e["groupsize"] = e["qweight"].repeat(1, times), e["g_idx"].repeat(times), 128 * times
    many = packed_linear_backward(g.to(DEV), e).view(T, times, 128)
    assert torch.equal(many, many[:, :1].expand_as(many))
    gd = g.double()
    want, mag = gd @ W, gd.abs() @ W.abs()
    assert_within(many[:, 0], want, sum_eps(R) * mag + ROUND[dtype] * want.abs() + TINY[dtype], "gx")


@pytest.mark.parametrize("T", [2, 40])
@pytest.mark.parametrize("D,I", [(4224, 40), (64, 8448)])
@pytest.mark.parametrize("nbits,groups", [(3, "128"), (4, "channel"), (5, "128"), (4, "32"), (4, "order128")])
def test_moe_many_chunks_a_wave(nbits, groups, D, I, T):
    """Experts of more chunks of 128 columns than waves share them, before the activation and after it."""
    dtype = (F16, BF16, F32)[(T + nbits) % 3]
    check_moe(*moe_case(T, T, D, I, 2, dtype, (nbits,) * 3, (groups,) * 3), 1, True)


@pytest.mark.parametrize("T", [6, 48])
@pytest.mark.parametrize("groups", ["128", "32", "order32"])
def test_moe_tokens_keep_to_themselves_to_the_bit(groups, T):
    """A NaN token sends itself to other experts, so the units' companions and their order change; the other
    tokens' results do not, to the last bit."""
    x, router, parts = moe_case(21, T, 256, 384, 6, BF16, groups=(groups,) * 3)
    x, router, args = x.to(DEV), router.to(DEV), [on(e, DEV) for e, _ in parts]
    clean = packed_moe(x, router, *args, 2)
    x[3, 3] = float("nan")
    y = packed_moe(x, router, *args, 2)
    assert bool(torch.isnan(y[3]).all())
    keep = [t for t in range(T) if t != 3]
    assert torch.equal(y[keep], clean[keep])


def test_moe_most_shared_memory():
    """The most units (64 tokens, each with 64 of 1024 experts) and the most scales a wave stages, of down along an
    order, leave least of the 160 KB."""
    check_moe(*moe_case(9, 64, 48, 62, 1024, BF16, (4, 4, 4), ("channel", "channel", "order1")), 64, True)
