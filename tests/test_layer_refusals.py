"""CPU tests of the layer-norm and 4-bit-weight entry points: what they refuse before any device is touched, and the
64-bit reference against itself."""
import ctypes as C

import pytest
import torch

from hpcdeepneuralnetworks_b200 import _lib, layer
from oracle import layer as ref

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -6
F32, BF16, F16 = 0, 1, 2


@pytest.fixture(scope="module")
def L(built_lib):
    return _lib.load()


def at(n):
    return C.c_void_p(n)


NULL = C.c_void_p(None)


def forward(L, rows=4, cols=8, eps=1e-5, type_=F32, x=at(0x1000), ldx=8, pt=F32, gamma=at(0x3000), beta=at(0x4000), y=at(0x2000), ldy=8,
            mean=NULL, rstd=NULL):
    return L.b2_layernorm(NULL, rows, cols, eps, type_, x, ldx, pt, gamma, beta, y, ldy, mean, rstd, NULL)


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(cols=0), dict(cols=-3), dict(cols=1 << 31, ldx=1 << 31, ldy=1 << 31), dict(ldx=7), dict(ldy=7), dict(type_=3),
    dict(type_=-1), dict(type_=BF16, pt=F16), dict(type_=F32, pt=BF16), dict(pt=9), dict(eps=-1e-9), dict(eps=float("nan")),
    dict(eps=float("inf")), dict(x=NULL), dict(y=NULL), dict(x=at(0x1002)), dict(gamma=at(0x3001)), dict(mean=at(0x5002)),
    dict(type_=F16, pt=F16, x=at(0x1001)), dict(y=at(0x1000), ldy=9), dict(y=at(0x1004)), dict(y=at(0x1000 + 3 * 32)),
])
def test_layernorm_refuses(L, bad):
    assert forward(L, **bad) == INVALID
    assert L.b2_last_error()


def test_layernorm_empty_is_a_no_op(L):
    assert forward(L, rows=0, x=NULL, y=NULL) == 0


def backward(L, rows=4, cols=8, type_=F32, dy=at(0x1000), lddy=8, x=at(0x2000), ldx=8, pt=F32, gamma=at(0x3000), mean=at(0x4000),
             rstd=at(0x5000), dx=at(0x6000), lddx=8, dg=at(0x7000), db=at(0x8000), ws=at(0x10000), nws=1 << 20):
    return L.b2_layernorm_backward(NULL, rows, cols, type_, dy, lddy, x, ldx, pt, gamma, mean, rstd, dx, lddx, dg, db, ws, nws, NULL)


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(cols=0), dict(lddy=7), dict(ldx=7), dict(lddx=7), dict(type_=5), dict(type_=BF16, pt=F16), dict(dy=NULL),
    dict(x=NULL), dict(mean=NULL), dict(rstd=NULL), dict(dx=at(0x6002)), dict(dg=at(0x7001)), dict(rstd=at(0x5001)),
    dict(dx=at(0x2000)), dict(dx=at(0x2010)), dict(dx=at(0x1000), lddx=9), dict(dx=at(0x1020)), dict(ws=at(0x10008)),
])
def test_layernorm_backward_refuses(L, bad):
    assert backward(L, **bad) == INVALID
    assert L.b2_last_error()


def test_layernorm_backward_workspace(L):
    need = L.b2_layernorm_backward_workspace_bytes(4, 8)
    assert need > 0
    assert backward(L, nws=need - 1) == WORKSPACE
    assert backward(L, ws=NULL) == WORKSPACE
    assert L.b2_layernorm_backward_workspace_bytes(0, 8) == 0
    assert backward(L, dx=NULL, dg=NULL, db=NULL, ws=NULL, nws=0) == 0          # nothing asked for


W4 = dict(N=4, K=64, group=32)


def quantize(L, N=4, K=64, group=32, type_=F32, W=at(0x1000), ldw=64, codes=at(0x8000), ldq=32, st=F32, scales=at(0x9000), zeros=NULL):
    return L.b2_w4_quantize(NULL, N, K, group, type_, W, ldw, codes, ldq, st, scales, zeros, NULL)


def dequantize(L, N=4, K=64, group=32, codes=at(0x8000), ldq=32, st=F32, scales=at(0x9000), zeros=NULL, type_=F32, W=at(0x1000), ldw=64,
               transpose=0):
    return L.b2_w4_dequantize(NULL, N, K, group, codes, ldq, st, scales, zeros, type_, W, ldw, transpose, NULL)


def matvec(L, M=2, N=4, K=64, group=32, alpha=1.0, type_=F32, x=at(0x1000), ldx=64, codes=at(0x8000), ldq=32, st=F32, scales=at(0x9000),
           zeros=NULL, beta=0.0, y=at(0x2000), ldy=4, ws=at(0x10000), nws=1 << 20):
    return L.b2_w4_matvec(NULL, M, N, K, group, alpha, type_, x, ldx, codes, ldq, st, scales, zeros, beta, y, ldy, ws, nws, NULL)


SHARED = [dict(N=-1), dict(K=-1), dict(group=0), dict(group=48), dict(group=512), dict(type_=3), dict(st=3), dict(ldq=31),
          dict(codes=NULL), dict(scales=NULL), dict(scales=at(0x9002)), dict(st=BF16, scales=at(0x9001)), dict(N=1 << 31)]


@pytest.mark.parametrize("bad", SHARED + [dict(ldw=63), dict(W=NULL), dict(W=at(0x1002)), dict(codes=at(0x1010))])
def test_w4_quantize_refuses(L, bad):
    assert quantize(L, **bad) == INVALID
    assert L.b2_last_error()


@pytest.mark.parametrize("bad", SHARED + [dict(ldw=63), dict(ldw=3, transpose=1), dict(W=NULL), dict(W=at(0x1001), type_=F16),
                                          dict(codes=at(0x1010))])
def test_w4_dequantize_refuses(L, bad):
    assert dequantize(L, **bad) == INVALID
    assert L.b2_last_error()


@pytest.mark.parametrize("bad", SHARED + [dict(M=-1), dict(ldx=63), dict(ldy=3), dict(x=NULL), dict(y=NULL), dict(x=at(0x1002)),
                                          dict(y=at(0x1000)), dict(y=at(0x1100)),
                                          dict(M=60, x=at(0x100000), y=at(0x200000), ws=at(0x10008))])
def test_w4_matvec_refuses(L, bad):
    assert matvec(L, **bad) == INVALID
    assert L.b2_last_error()


def test_w4_matvec_refuses_many_rows(L):
    assert matvec(L, M=layer.W4_MAX_ROWS + 1) == UNSUPPORTED
    assert b"b2_w4_dequantize" in L.b2_last_error()


def test_w4_matvec_refuses_the_longest_rows(L):
    K = 2 ** 27 + 1
    assert matvec(L, K=K, ldx=K, ldq=K) == UNSUPPORTED
    assert L.b2_w4_matvec_workspace_bytes(60, 4, K, BF16) == 0 < L.b2_w4_matvec_workspace_bytes(60, 4, K - 1, BF16)


def test_w4_matvec_workspace(L):
    for type_ in (F32, BF16, F16):
        need = L.b2_w4_matvec_workspace_bytes(60, 4, 64, type_)
        assert need > 0
        rows = dict(M=60, type_=type_, x=at(0x100000), y=at(0x200000))
        assert matvec(L, nws=need - 1, **rows) == WORKSPACE
        assert matvec(L, ws=NULL, **rows) == WORKSPACE
        assert L.b2_w4_matvec_workspace_bytes(1, 4, 64, type_) == 0        # a small product needs none
    assert L.b2_w4_matvec_workspace_bytes(0, 4, 64, F32) == 0 and L.b2_w4_matvec_workspace_bytes(60, 4, 0, F32) == 0
    assert L.b2_w4_matvec_workspace_bytes(60, 4, 64, 7) == 0


def test_w4_empty_calls_are_no_ops(L):
    assert quantize(L, N=0, W=NULL, codes=NULL, scales=NULL) == 0
    assert quantize(L, K=0, ldw=0, ldq=0, W=NULL, codes=NULL, scales=NULL) == 0
    assert dequantize(L, N=0, W=NULL, codes=NULL, scales=NULL) == 0
    assert matvec(L, M=0, x=NULL, y=NULL) == 0
    assert matvec(L, N=0, ldy=0, codes=NULL, scales=NULL, y=NULL) == 0


def test_python_wrappers_refuse_host_tensors_and_wrong_groups(built_lib):
    t = torch.zeros(4, 8)
    with pytest.raises(TypeError, match="expected a CUDA tensor"):
        layer.layernorm(4, 8, 1e-5, t, None, None, t)
    with pytest.raises(TypeError, match="expected a CUDA tensor"):
        layer.layernorm_backward(4, 8, t, t, None, t, t, t, None, None)
    with pytest.raises(TypeError, match="expected a CUDA tensor"):
        layer.w4_quantize(4, 8, 32, t, t, t)
    with pytest.raises(TypeError, match="expected a CUDA tensor"):
        layer.w4_dequantize(4, 8, 32, t, t)
    with pytest.raises(TypeError, match="expected a CUDA tensor"):
        layer.w4_matvec(4, 8, 8, 32, 1.0, t, t, t, None, 0.0)
    with pytest.raises(ValueError, match="group 48"):
        layer.w4_empty(4, 8, 48)


class FakeCuda(torch.Tensor):
    """A host tensor that says it lies on CUDA device 0: enough for the checks that come before any device work."""

    is_cuda = True

    def get_device(self):
        return 0


def fake(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(FakeCuda)


def test_matrix_checks():
    m = layer._matrix
    t = fake(4, 16)
    assert m(t, 4, 16, None, "t", 0) == (t.data_ptr(), 16)
    assert m(t[:, :8], 4, 8, None, "t", 0) == (t.data_ptr(), 16)            # a column slice keeps its pitch
    assert m(t[:, 8:], 3, 8, None, "t", 0) == (t.data_ptr() + 32, 16)
    assert m(fake(64), 4, 16, None, "t", 0)[1] == 16                       # flat memory
    assert m(fake(2, 2, 16), 4, 16, None, "t", 0)[1] == 16                 # leading dimensions together
    assert m(t, 4, 8, 16, "t", 0)[1] == 16
    for bad in (lambda: m(t, 4, 8, None, "t", 0),                           # rows are not 8 long
                lambda: m(t, 5, 16, None, "t", 0), lambda: m(fake(63), 4, 16, None, "t", 0),
                lambda: m(t.t(), 16, 4, None, "t", 0), lambda: m(t[:, ::2], 4, 8, None, "t", 0),
                lambda: m(t, 5, 8, 16, "t", 0), lambda: m(t[:, 8:], 4, 16, 16, "t", 0), lambda: m(t[:, :8], 5, 8, None, "t", 0),
                lambda: m(t, 4, 16, None, "t", 1)):                        # another device is current
        with pytest.raises(ValueError):
            bad()


def test_reference_gradients_agree_with_differences():
    g = torch.Generator().manual_seed(3)
    x, dy = torch.randn(3, 7, generator=g, dtype=torch.float64), torch.randn(3, 7, generator=g, dtype=torch.float64)
    gamma, beta = torch.randn(7, generator=g, dtype=torch.float64), torch.randn(7, generator=g, dtype=torch.float64)
    y, mean, rstd, _ = ref.layernorm(x, gamma, beta, 1e-5)
    dx, dgamma, dbeta, _ = ref.layernorm_backward(dy, x, gamma, mean, rstd)
    loss = lambda x_, g_, b_: float((ref.layernorm(x_, g_, b_, 1e-5)[0] * dy).sum())  # noqa: E731
    e = 1e-6
    for what, grad in (("x", dx), ("gamma", dgamma), ("beta", dbeta)):
        base = {"x": x, "gamma": gamma, "beta": beta}[what]
        for i in range(base.numel()):
            up, down = base.clone(), base.clone()
            up.view(-1)[i] += e
            down.view(-1)[i] -= e
            args = lambda t: [t if n == what else v for n, v in (("x", x), ("gamma", gamma), ("beta", beta))]  # noqa: E731
            assert abs((loss(*args(up)) - loss(*args(down))) / (2 * e) - float(grad.view(-1)[i])) < 1e-6


def test_reference_packing_round_trip():
    g = torch.Generator().manual_seed(4)
    for K in (1, 2, 33, 64):
        codes = torch.randint(0, 16, (5, K), generator=g)
        packed = ref.w4_pack(codes)
        assert packed.shape == (5, (K + 1) // 2)
        assert torch.equal(ref.w4_unpack(packed, K), codes)
        if K % 2:
            assert int((packed[:, -1] >> 4).max()) == 0
    W = torch.randn(6, 100, generator=g)
    codes, scales, zeros = ref.w4_quantize(W, 32, torch.float32, True)
    off = (ref.w4_values(codes, scales, zeros, 32) - W.double()).abs()
    # a code is off by half a step, and by up to half a step more where the zero point was rounded and the code clamped
    assert bool((off <= 1.001 * scales.double()[:, torch.arange(100) // 32]).all())


def test_short_calls_leave_everything_unusual_to_the_checks(built_lib):
    """The extension answers False to what it does not know, whatever that is, and never calls the library for it."""
    layer._load()
    quick, t, i = layer._quick, torch.zeros(4, 8), 2 ** 70
    for name, count in (("layernorm", 10), ("layernorm_backward", 12), ("w4_quantize", 8), ("w4_dequantize", 9), ("w4_matvec", 13)):
        f = getattr(quick, name)
        for args in ([], [None] * (count - 1), [None] * count, [t] * count, [1] * count, [None] + [i] * (count - 1), ["x"] * count,
                     [None] + [4] * 3 + [t] * (count - 4), [object()] + [4, 8] + [fake(4, 8)] * (count - 3)):
            assert f(*args) is False, (name, args)
    for args in ((), (1,) * 8, ({},) + ("x",) * 7):
        with pytest.raises(TypeError):
            quick.bind(*args)
