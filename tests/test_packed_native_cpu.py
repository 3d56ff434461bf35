"""The packed products' and the scoring's C entries and Python checks, without a device: bad arguments are
refused before any launch, sizes of workspaces, entries on the CPU."""
import ctypes

import pytest
import torch

import gptq_plus_mp_quant_amd as G
from gptq_plus_mp_quant_amd import _native as nat
from gptq_plus_mp_quant_amd import kernels as K
from tests._packed import make_entry

FAKE, NULL = 16, None


def _lib():
    if not nat.LIB_PATH.exists():
        pytest.skip("library not built")
    return nat.load()


LINEAR = dict(x=FAKE, dtype=nat.RQ_F16, T=1, ldx=64, C=64, q=FAKE, ldp=8, nbits=4, R=32, scales=FAKE, lds=32, ngroups=2, g_idx=NULL,
              groupsize=32)
LINEAR_BAD = [dict(T=-1), dict(x=NULL), dict(ldx=63), dict(C=0), dict(q=NULL), dict(ldp=7), dict(nbits=1), dict(nbits=10),
              dict(R=0), dict(scales=NULL), dict(lds=31), dict(ngroups=0), dict(groupsize=0), dict(groupsize=-32), dict(groupsize=31),
              dict(dtype=7)]


@pytest.mark.parametrize("bad", LINEAR_BAD, ids=str)
def test_packed_linear_refusals(bad):
    a = list({**LINEAR, **bad}.values())
    lib = _lib()
    assert lib.rq_packed_linear(*a, NULL, FAKE, 32, NULL) == nat.RQ_EINVAL
    if "ldx" not in bad:                       # the gradient's row stride belongs to the R side
        a[3] = 32
        assert lib.rq_packed_linear_grad(*a, FAKE, 64, FAKE, 1 << 30, NULL) == nat.RQ_EINVAL


def test_packed_linear_outputs():
    a, lib = list(LINEAR.values()), _lib()
    assert lib.rq_packed_linear(*a, NULL, NULL, 32, NULL) == nat.RQ_EINVAL
    assert lib.rq_packed_linear(*a, NULL, FAKE, 31, NULL) == nat.RQ_EINVAL
    g = list({**LINEAR, "ldx": 32}.values())
    assert lib.rq_packed_linear_grad(*g, NULL, 64, FAKE, 1 << 30, NULL) == nat.RQ_EINVAL
    assert lib.rq_packed_linear_grad(*g, FAKE, 63, FAKE, 1 << 30, NULL) == nat.RQ_EINVAL
    assert lib.rq_packed_linear_grad(*g, FAKE, 64, NULL, 0, NULL) == nat.RQ_EINVAL
    g[3] = 31
    assert lib.rq_packed_linear_grad(*g, FAKE, 64, FAKE, 1 << 30, NULL) == nat.RQ_EINVAL
    # no tokens: nothing is read, nothing is launched
    z = list({**LINEAR, "T": 0, "x": NULL}.values())
    assert lib.rq_packed_linear(*z, NULL, NULL, 32, NULL) == nat.RQ_OK
    assert lib.rq_packed_linear_grad(*z, NULL, 64, NULL, 0, NULL) == nat.RQ_OK


@pytest.mark.parametrize("T", [1, 16, 63, 64, 65, 100, 129])
def test_gradient_workspace_holds_every_launch(T):
    """Tokens go in launches of 64; a shorter last one may be cut into more parts."""
    lib = _lib()
    for R, C in ((32, 64), (4096, 4096), (14336, 128), (100, 28672)):
        need = lib.rq_packed_linear_grad_workspace_bytes(T, R, C)
        assert need >= lib.rq_packed_linear_grad_workspace_bytes(min(T, 64), R, C) >= 4 * min(T, 64) * C
        if T > 64 and T % 64:
            assert need >= lib.rq_packed_linear_grad_workspace_bytes(T % 64, R, C)
    assert lib.rq_packed_linear_grad_workspace_bytes(0, 32, 64) == 0
    for bad in ((-1, 32, 64), (1, 0, 64), (1, 32, 0)):
        assert lib.rq_packed_linear_grad_workspace_bytes(*bad) < 0


def _experts(**over):
    f = {**dict(qweight=FAKE, scales=FAKE, g_idx=None, ldp=8, lds=64, stride_q=512, stride_scales=128, nbits=4, ngroups=2,
                groupsize=32), **over}
    return nat.PackedExperts(*(f[n] for n, _ in nat.PackedExperts._fields_))


MOE = dict(x=FAKE, dtype=nat.RQ_BF16, T=2, ldx=64, D=64, router=FAKE, ldr=64, E=4, K=2, norm=1, I=64)


@pytest.mark.parametrize("bad", [dict(T=-1), dict(x=NULL), dict(ldx=63), dict(D=0), dict(router=NULL), dict(ldr=63), dict(E=0),
                                 dict(E=1025), dict(K=0), dict(K=5), dict(E=100, K=65), dict(I=0), dict(dtype=9)], ids=str)
def test_packed_moe_refusals(bad):
    a, w, lib = list({**MOE, **bad}.values()), _experts(), _lib()
    ws = lib.rq_packed_moe_workspace_bytes(2, 64, 64, 4, 2)
    assert ws > 0
    refs = [ctypes.byref(w)] * 3
    assert lib.rq_packed_moe(*a, *refs, FAKE, 64, NULL, NULL, FAKE, 1 << 40, NULL) == nat.RQ_EINVAL


def test_packed_moe_experts_and_outputs():
    a, lib, ok = list(MOE.values()), _lib(), _experts()
    need = lib.rq_packed_moe_workspace_bytes(2, 64, 64, 4, 2)

    def call(weights, y=FAKE, ldy=64, ws=FAKE, nbytes=need):
        return lib.rq_packed_moe(*a, *(None if w is None else ctypes.byref(w) for w in weights), y, ldy, NULL, NULL, ws, nbytes, NULL)

    for i in range(3):
        for bad in (None, _experts(qweight=None), _experts(scales=None), _experts(ldp=7), _experts(lds=63), _experts(nbits=1),
                    _experts(ngroups=0), _experts(groupsize=0), _experts(groupsize=16)):
            weights = [ok, ok, ok]
            weights[i] = bad
            assert call(weights) == nat.RQ_EINVAL
    assert call([ok] * 3, y=NULL) == call([ok] * 3, ldy=63) == nat.RQ_EINVAL
    assert call([ok] * 3, ws=NULL) == call([ok] * 3, nbytes=need - 1) == nat.RQ_EINVAL
    a[2] = 0
    assert call([ok] * 3) == nat.RQ_OK
    # a workspace serves 64 tokens at a time
    assert lib.rq_packed_moe_workspace_bytes(64, 64, 64, 4, 2) == lib.rq_packed_moe_workspace_bytes(1000, 64, 64, 4, 2)


SCORE = dict(z=FAKE, dtype=nat.RQ_F32, N=1, ldz=100, V=100, targets=FAKE, ignore=-100, top=5)


@pytest.mark.parametrize("bad", [dict(N=-1), dict(z=NULL), dict(ldz=99), dict(V=0), dict(V=(1 << 30) + 1, ldz=1 << 31),
                                 dict(targets=NULL), dict(top=-1), dict(top=65), dict(V=4, top=5), dict(dtype=5)], ids=str)
def test_token_logprobs_refusals(bad):
    a = list({**SCORE, **bad}.values())
    assert _lib().rq_token_logprobs(*a, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, NULL) == nat.RQ_EINVAL


def test_token_logprobs_outputs_and_workspace():
    lib, a = _lib(), list(SCORE.values())
    for i in range(5):
        out = [FAKE] * 5
        out[i] = NULL
        assert lib.rq_token_logprobs(*a, *out, FAKE, 1 << 40, NULL) == nat.RQ_EINVAL
    big = list({**SCORE, "V": 128256, "ldz": 128256}.values())
    need = lib.rq_token_logprobs_workspace_bytes(1, 128256, 5)
    assert need > 0
    assert lib.rq_token_logprobs(*big, *[FAKE] * 5, FAKE, need - 1, NULL) == nat.RQ_EINVAL
    assert lib.rq_token_logprobs(*big, *[FAKE] * 5, NULL, need, NULL) == nat.RQ_EINVAL
    assert lib.rq_token_logprobs_workspace_bytes(0, 100, 5) == lib.rq_token_logprobs_workspace_bytes(4096, 128256, 5) == 0
    for bad in ((-1, 100, 5), (1, 0, 0), (1, 4, 5), (1, 100, 65)):
        assert lib.rq_token_logprobs_workspace_bytes(*bad) < 0
    g = [FAKE, nat.RQ_F32, 1, 100, 100, FAKE, -100, FAKE, FAKE, NULL, FAKE, 100, NULL]
    for i, v in ((0, NULL), (1, 5), (2, -1), (3, 99), (4, 0), (5, NULL), (7, NULL), (8, NULL), (10, NULL), (11, 99)):
        assert lib.rq_token_logprobs_grad(*g[:i], v, *g[i + 1:]) == nat.RQ_EINVAL


def test_cpu_tensors_are_refused():
    e, _ = make_entry(0, 16, 64, 4, "32")
    with pytest.raises(RuntimeError):
        G.packed_linear(torch.zeros(1, 64), e)
    with pytest.raises(RuntimeError):
        G.packed_linear_backward(torch.zeros(1, 16), e)
    with pytest.raises(RuntimeError):
        G.stack_packed([e])
    with pytest.raises(RuntimeError):
        G.token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))


def test_operands_that_are_no_tensors_are_refused():
    """With the errors that wrong tensors get, not an AttributeError."""
    e, _ = make_entry(0, 16, 64, 4, "32")
    for call in (lambda: G.packed_linear([0.0] * 64, e), lambda: G.packed_linear_backward([0.0] * 16, e),
                 lambda: G.packed_moe(torch.zeros(1, 64), None, e, e, e, 1),
                 lambda: G.token_logprobs_backward(None, None, None, None)):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            call()


@pytest.fixture
def two_devices(monkeypatch):
    """A library that records the current device of every call, on a host with device 0 current of two."""
    seen, current = [], [0]

    class Library:
        def __getattr__(self, name):
            def entry(*args):
                seen.append((name, current[0], args[-1].value if isinstance(args[-1], ctypes.c_void_p) else args[-1]))
                return nat.RQ_OK
            return entry

    class On:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    monkeypatch.setattr(nat, "load", lambda: Library())
    monkeypatch.setattr(nat, "_raw_stream_of", lambda index: 100 + index)
    monkeypatch.setattr(nat, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d: type("S", (), dict(cuda_stream=100 + d.index, device=d)))
    return seen


@pytest.mark.parametrize("index", [0, 1])
def test_kernels_go_to_the_tensors_device(two_devices, index):
    """A call on tensors of a device that is not current makes it current for the launch (a default stream's handle
    is 0 on every device), and leaves the current one as it was."""
    class T:
        device = torch.device("cuda", index)

        def get_device(self):
            return index

    @nat.on_device_of_first
    def product(t, n):
        """Twice the number."""
        nat.check("rq_packed_linear", nat.load().rq_packed_linear(n, nat.raw_stream(t)))
        return 2 * n

    assert product(T(), 4) == 8 and product.__doc__ == "Twice the number."
    nat.call("rq_find_params", 1, nat.stream_of(T.device))
    nat.call("rq_hessian_math", 0)
    assert two_devices == [("rq_packed_linear", index, 100 + index), ("rq_find_params", index, 100 + index), ("rq_hessian_math", 0, 0)]
    assert nat._current_device() == 0
    with pytest.raises(ZeroDivisionError):
        nat.on_device_of_first(lambda t: 1 // 0)(T())
    assert nat._current_device() == 0
    # the wrappers of the packed operators and of scoring are made so
    for fn in (K.packed_linear, K.packed_linear_grad, K.packed_moe, K.token_logprobs, K.token_logprobs_grad):
        assert fn.__wrapped__
