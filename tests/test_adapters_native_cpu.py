"""The C entries and Python checks of the adapters, the gated block and the distillation loss, without a device: bad
arguments are refused before any launch, sizes of workspaces, tensors on the CPU."""
import pytest
import torch

import gptq_plus_mp_quant_amd as G
from gptq_plus_mp_quant_amd import _native as nat
from gptq_plus_mp_quant_amd import adapters as A
from gptq_plus_mp_quant_amd import distillation as D
from gptq_plus_mp_quant_amd import kernels as K
from gptq_plus_mp_quant_amd import packed as P
from tests._packed import make_entry

FAKE, NULL, MUCH = 16, None, 1 << 50


def _lib():
    if not nat.LIB_PATH.exists():
        pytest.skip("library not built")
    return nat.load()


def _call(entry, base, **over):
    return getattr(_lib(), entry)(*{**base, **over}.values())


LORA = dict(x=FAKE, dtype=nat.RQ_F16, T=3, ldx=64, C=64, q=FAKE, ldp=8, nbits=4, R=32, scales=FAKE, lds=32, ngroups=2, g_idx=NULL,
            groupsize=32, bias=NULL, a=FAKE, b=FAKE, n=2, r=4, ids=FAKE, scaling=NULL, scale=1.0, y=FAKE, ldy=32, ws=FAKE,
            nbytes=MUCH, stream=NULL)
WEIGHT_BAD = [dict(q=NULL), dict(ldp=7), dict(nbits=1), dict(nbits=10), dict(R=0), dict(C=0), dict(scales=NULL), dict(lds=31),
              dict(ngroups=0), dict(groupsize=0), dict(groupsize=-32), dict(groupsize=31)]
ADAPTER_BAD = [dict(a=NULL), dict(b=NULL), dict(n=0), dict(n=65536), dict(r=0), dict(r=257), dict(T=-1), dict(T=(1 << 19) + 1),
               dict(dtype=7), dict(x=NULL), dict(ldx=63), dict(ws=NULL), dict(nbytes=0)]


@pytest.mark.parametrize("bad", WEIGHT_BAD + ADAPTER_BAD + [dict(y=NULL), dict(ldy=31)], ids=str)
def test_lora_refusals(bad):
    assert _call("rq_packed_linear_lora", LORA, **bad) == nat.RQ_EINVAL


LORA_GRAD = dict(gy=FAKE, dtype=nat.RQ_F16, T=1, ldg=32, x=FAKE, ldx=64, C=64, q=FAKE, ldp=8, nbits=4, R=32, scales=FAKE, lds=32,
                 ngroups=2, g_idx=NULL, groupsize=32, a=FAKE, b=FAKE, n=2, r=4, ids=FAKE, scaling=NULL, scale=1.0, gx=FAKE, ldgx=64,
                 ga=FAKE, gb=FAKE, ws=FAKE, nbytes=MUCH, stream=NULL)


@pytest.mark.parametrize("bad", WEIGHT_BAD + ADAPTER_BAD + [dict(gy=NULL), dict(ldg=31), dict(ldgx=63), dict(ga=NULL), dict(gb=NULL)],
                         ids=str)
def test_lora_gradient_refusals(bad):
    assert _call("rq_packed_linear_lora_grad", LORA_GRAD, **bad) == nat.RQ_EINVAL


def test_lora_workspaces_and_empty_calls():
    lib = _lib()
    assert _call("rq_packed_linear_lora", LORA, T=0, x=NULL, y=NULL, ws=NULL, nbytes=0) == nat.RQ_OK
    for T in (1, 16, 63, 64, 65, 100, 1000):
        for R, C, r in ((32, 64, 1), (4096, 14336, 64), (100, 28672, 256)):
            need = lib.rq_packed_linear_lora_workspace_bytes(T, R, C, r, nat.RQ_F16)
            assert need >= 4 * T * r or (need == 0 and T == r == 1)            # one token of few ranks needs none
            grad = lib.rq_packed_linear_lora_grad_workspace_bytes(T, R, C, r)
            assert grad >= 8 * T * r + 4 * min(T, 64) * C
            size = dict(T=T, C=C, ldx=C, R=R, ldp=C, lds=R, groupsize=C, r=r)
            assert need == 0 or _call("rq_packed_linear_lora", LORA, **size, ldy=R, nbytes=need - 1) == nat.RQ_EINVAL
            assert _call("rq_packed_linear_lora_grad", LORA_GRAD, **size, ldg=R, ldgx=C, nbytes=grad - 1) == nat.RQ_EINVAL
    for T, C, r in ((-1, 64, 4), (1, 0, 4), (1, 64, 0), (1, 64, 257), ((1 << 19) + 1, 64, 4), (1, 1 << 30, 256)):
        assert lib.rq_packed_linear_lora_workspace_bytes(T, 32, C, r, nat.RQ_F16) < 0
    assert lib.rq_packed_linear_lora_workspace_bytes(1, 0, 64, 4, nat.RQ_F16) < 0
    assert lib.rq_packed_linear_lora_workspace_bytes(1, 32, 64, 4, 7) < 0
    for bad in ((-1, 32, 64, 4), (1, 0, 64, 4), (1, 32, 0, 4), (1, 32, 64, 0), (1, 1 << 30, 64, 256)):
        assert lib.rq_packed_linear_lora_grad_workspace_bytes(*bad) < 0


def _weight(**over):
    f = {**dict(qweight=FAKE, scales=FAKE, g_idx=0, ldp=8, lds=32, nbits=4, ngroups=2, groupsize=32), **over}
    return nat.PACKED_WEIGHT.pack(*(v or 0 for v in f.values()))


def _gated(gate=_weight(), up=_weight(), **over):
    base = dict(x=FAKE, dtype=nat.RQ_BF16, T=1, ldx=64, C=64, I=32, gate=gate, up=up, act=0,
                pre=NULL, h=FAKE, ldh=32, ws=NULL, nbytes=0, stream=NULL)
    return _call("rq_packed_gated", base, **over)


def _gated_grad(gate=_weight(), up=_weight(), **over):
    base = dict(gh=FAKE, dtype=nat.RQ_BF16, T=1, ldg=32, I=32, pre=FAKE, act=0, gate=gate, up=up, C=64, gx=FAKE, ldx=64, ws=FAKE, nbytes=MUCH, stream=NULL)
    return _call("rq_packed_gated_grad", base, **over)


BOTH_BAD = [dict(T=-1), dict(T=(1 << 19) + 1), dict(dtype=9), dict(C=0), dict(I=0), dict(act=-1), dict(act=3), dict(ldx=63)]
BAD_WEIGHTS = [None, _weight(qweight=None), _weight(scales=None), _weight(ldp=7), _weight(lds=31), _weight(nbits=1), _weight(nbits=10),
               _weight(ngroups=0), _weight(groupsize=0), _weight(groupsize=31), _weight(groupsize=-32)]


def test_gated_refusals():
    for bad in BOTH_BAD + [dict(x=NULL), dict(h=NULL), dict(ldh=31)]:
        assert _gated(**bad) == nat.RQ_EINVAL, bad
    for bad in BOTH_BAD + [dict(gh=NULL), dict(pre=NULL), dict(gx=NULL), dict(ldg=31), dict(ws=NULL), dict(nbytes=0)]:
        assert _gated_grad(**bad) == nat.RQ_EINVAL, bad
    for w in BAD_WEIGHTS:
        assert _gated(gate=w) == _gated(up=w) == _gated_grad(gate=w) == _gated_grad(up=w) == nat.RQ_EINVAL
    # weights of different bits go by way of both products
    assert _gated(up=_weight(nbits=3)) == nat.RQ_EINVAL
    assert _gated(T=0, x=NULL, h=NULL) == _gated_grad(T=0, gh=NULL, pre=NULL, gx=NULL, ws=NULL, nbytes=0) == nat.RQ_OK


def test_gated_workspaces():
    lib = _lib()

    def need(T, gate, up, I=32, C=64, dtype=nat.RQ_BF16):
        return lib.rq_packed_gated_workspace_bytes(T, I, C, dtype, gate, up)

    assert need(5, _weight(), _weight()) == 0
    assert need(5, _weight(), _weight(nbits=3)) == 5 * 2 * 32 * 4
    assert need(5, _weight(), _weight(ngroups=1, groupsize=0)) == 5 * 2 * 32 * 4
    # more tokens than a tile: x once more, whole tiles of 16 and chunks of 128, where a weight's groups are runs of 128
    whole = _weight(ngroups=1, groupsize=0)              # C = 64, one chunk
    assert need(17, whole, whole) == 32 * 128 * 2 and need(17, whole, whole, dtype=nat.RQ_F32) == 32 * 128 * 6
    assert need(16, whole, whole) == need(17, _weight(), _weight()) == 0
    assert _gated(whole, whole, T=17, ws=FAKE, nbytes=32 * 128 * 2 - 1) == nat.RQ_EINVAL
    assert need(1, whole, whole, dtype=7) < 0
    assert need(-1, _weight(), _weight()) < 0 and need(1, _weight(), _weight(ldp=7)) < 0 and need(1, _weight(), _weight(), I=0) < 0
    for T in (1, 63, 64, 65, 100, 200):
        for I, C in ((32, 64), (14336, 4096), (100, 8192)):
            grad = lib.rq_packed_gated_grad_workspace_bytes(T, I, C)
            assert grad >= 4 * (min(T, 64) * 2 * I + 2 * min(T, 64) * C)
            w = _weight(ldp=C, lds=I, groupsize=C)
            assert _gated_grad(w, w, T=T, I=I, ldg=I, C=C, ldx=C, nbytes=grad - 1) == nat.RQ_EINVAL
    for bad in ((-1, 32, 64), (1, 0, 64), (1, 32, 0), ((1 << 19) + 1, 32, 64)):
        assert lib.rq_packed_gated_grad_workspace_bytes(*bad) < 0


DISTILL = dict(z=FAKE, dtype=nat.RQ_F32, N=1, ldz=100, V=100, ids=FAKE, t=FAKE, K=5, temperature=1.0, tail=1)
DISTILL_BAD = [dict(N=-1), dict(z=NULL), dict(ldz=99), dict(V=0), dict(V=(1 << 30) + 1, ldz=1 << 31), dict(ids=NULL), dict(t=NULL),
               dict(K=0), dict(K=257), dict(temperature=0.0), dict(temperature=2.0), dict(temperature=float("nan"), tail=0),
               dict(temperature=1e7, tail=0), dict(temperature=-1.0, tail=0), dict(tail=2), dict(tail=-1), dict(dtype=5)]


@pytest.mark.parametrize("bad", DISTILL_BAD, ids=str)
def test_distillation_refusals(bad):
    a = list({**DISTILL, **bad}.values())
    assert _lib().rq_distill_loss(*a, FAKE, FAKE, FAKE, MUCH, NULL) == nat.RQ_EINVAL
    assert _lib().rq_distill_loss_grad(*a, FAKE, FAKE, FAKE, 1 << 40, NULL) == nat.RQ_EINVAL


def test_distillation_outputs_and_workspace():
    lib, a = _lib(), list(DISTILL.values())
    assert lib.rq_distill_loss(*a, NULL, FAKE, FAKE, MUCH, NULL) == lib.rq_distill_loss(*a, FAKE, NULL, FAKE, MUCH, NULL) == nat.RQ_EINVAL
    for out in ((NULL, FAKE, FAKE, 100), (FAKE, NULL, FAKE, 100), (FAKE, FAKE, NULL, 100), (FAKE, FAKE, FAKE, 99)):
        assert lib.rq_distill_loss_grad(*a, *out, NULL) == nat.RQ_EINVAL
    big = list({**DISTILL, "V": 128256, "ldz": 128256}.values())
    need = lib.rq_distill_loss_workspace_bytes(1, 128256)
    assert need > 0
    assert lib.rq_distill_loss(*big, FAKE, FAKE, FAKE, need - 1, NULL) == lib.rq_distill_loss(*big, FAKE, FAKE, NULL, need, NULL) == nat.RQ_EINVAL
    assert lib.rq_distill_loss_workspace_bytes(0, 100) == lib.rq_distill_loss_workspace_bytes(4096, 128256) == 0
    for bad in ((-1, 100), (1, 0), (1, (1 << 30) + 1)):
        assert lib.rq_distill_loss_workspace_bytes(*bad) < 0
    none = list({**DISTILL, "N": 0, "z": NULL, "ids": NULL, "t": NULL}.values())
    assert lib.rq_distill_loss(*none, NULL, NULL, NULL, 0, NULL) == lib.rq_distill_loss_grad(*none, NULL, NULL, NULL, 100, NULL) == nat.RQ_OK


def test_cpu_tensors_and_what_is_no_tensor_are_refused():
    e, _ = make_entry(0, 16, 64, 4, "32")
    x, a, b = torch.zeros(1, 64), torch.zeros(1, 2, 64), torch.zeros(1, 16, 2)
    z, ids, t = torch.zeros(2, 8), torch.zeros((2, 3), dtype=torch.int64), torch.zeros(2, 3)
    for call in (lambda: G.packed_linear_lora(x, e, a, b), lambda: G.packed_linear_lora_backward(x[:, :16], x, e, a, b),
                 lambda: G.packed_gated(x, e, e), lambda: G.packed_gated_backward(x[:, :16], torch.zeros(1, 2, 16), e, e),
                 lambda: G.distillation_loss(z, ids, t), lambda: G.distillation_loss_backward(z, ids, t, torch.zeros(2, 8), t[:, 0])):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: G.packed_linear_lora([0.0] * 64, e, None, None), lambda: G.packed_linear_lora_backward(None, None, e, a, b),
                 lambda: G.packed_gated(None, e, e), lambda: G.packed_gated_backward(None, None, e, e),
                 lambda: G.distillation_loss(None, None, None), lambda: G.distillation_loss_backward(None, None, None, None, None)):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            call()


def test_wrappers_go_to_the_tensors_device():
    for fn in (K.packed_linear_lora, K.packed_linear_lora_grad, K.packed_gated, K.packed_gated_grad, K.distill_loss, K.distill_loss_grad):
        assert fn.__wrapped__


def test_autograd_checks_what_needs_a_gradient_on_any_device():
    e, _ = make_entry(0, 16, 64, 4, "32")
    with pytest.raises(RuntimeError):
        G.packed_linear_lora(torch.zeros(1, 64, requires_grad=True), e, torch.zeros(1, 2, 64), torch.zeros(1, 16, 2))
    with pytest.raises(RuntimeError):
        G.distillation_loss(torch.zeros(2, 8, requires_grad=True), torch.zeros((2, 3), dtype=torch.int64), torch.zeros(2, 3))


class _Drops(torch.autograd.Function):
    """Passes on no gradient."""
    @staticmethod
    def forward(ctx, x):
        return x.clone()

    @staticmethod
    def backward(ctx, g):
        return None


def _stand_ins(monkeypatch):
    """The gated block and the loss with the launches left out, as (Function, arguments, leaf), and what their backward is given."""
    e, seen = make_entry(0, 16, 64, 4, "32")[0], []
    monkeypatch.setattr(P, "_gated", lambda x, *a: (x[:, :16].clone(), x.new_zeros((2, 2, 16))))
    monkeypatch.setattr(P, "_gated_backward", lambda g, *a: g.new_ones((2, 64)))
    monkeypatch.setattr(D, "_forward", lambda z, *a: D.Distillation(z.sum(-1), z.new_zeros((2, 8))))
    monkeypatch.setattr(D, "_backward", lambda z, *a: torch.ones_like(z))
    x, z = torch.zeros((2, 64), requires_grad=True), torch.zeros((2, 8), requires_grad=True)
    ids, t = torch.zeros((2, 3), dtype=torch.int64), torch.zeros((2, 3))
    for cls in (P._PackedGated, D._DistillationLoss):
        def backward(ctx, *grads, real=cls.backward):
            seen.append(grads)
            return real(ctx, *grads)
        monkeypatch.setattr(cls, "backward", staticmethod(backward))
    return ((P._PackedGated, (x, e, e, "silu"), x), (D._DistillationLoss, (z, ids, t, 1.0, "bucket"), z)), seen


def test_no_zeros_are_filled_for_what_takes_no_gradient(monkeypatch):
    """pre and the statistics are results without a gradient: none is made for them on the way back, and none of the
    input where the result's own is missing."""
    cases, seen = _stand_ins(monkeypatch)
    for fn, args, leaf in cases:
        fn.apply(*args)[0].sum().backward()
        assert seen[-1][0] is not None and seen[-1][1] is None and bool((leaf.grad == 1).all())
        leaf.grad = None
        _Drops.apply(fn.apply(*args)[0]).sum().backward()
        assert leaf.grad is None


def test_constants_made_in_inference_mode_have_a_backward_pass(monkeypatch):
    """A teacher's list, a frozen part's activations, another's adapters: what needs no gradient may come from there, and
    what is changed in place between the passes is still noticed."""
    (_, (dist, (z, *_), _)), _ = _stand_ins(monkeypatch)
    e = make_entry(0, 16, 64, 4, "32")[0]
    monkeypatch.setattr(A, "_forward", lambda x, *a: x[:, :16] * 1)
    monkeypatch.setattr(A, "_backward", lambda *a: (torch.ones(2, 64), torch.ones(1, 2, 64), torch.ones(1, 16, 2)))
    with torch.inference_mode():
        ids, t = torch.zeros((2, 3), dtype=torch.int64), torch.zeros((2, 3))
        x, b, s = torch.zeros((2, 64)), torch.zeros((1, 16, 2)), torch.ones(1)
        inferred = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in e.items()}
    dist.apply(z, ids, t, 1.0, "bucket")[0].sum().backward()
    assert bool((z.grad == 1).all())
    leaf = torch.zeros((1, 2, 64), requires_grad=True)
    for entry in (e, inferred):
        leaf.grad = None
        A._PackedLinearLora.apply(x, leaf, b, entry, None, s, None).sum().backward()
        assert bool((leaf.grad == 1).all())
        y = A._PackedLinearLora.apply(x, leaf, b, entry, None, s, None).sum()
        with torch.no_grad():
            leaf.add_(1)
        with pytest.raises(RuntimeError):
            y.backward()
