"""What becomes of a status that a layer operator's call ends with: refusals are worded by the checks in Python, every other
error reaches the caller once, and no call is made a second time after work may have been enqueued."""
import ctypes as C

import pytest
import torch

from hpcdeepneuralnetworks_b200 import _lib, layer
from hpcdeepneuralnetworks_b200.blas import _default

CUDA, TIMEOUT = -3, -4
NAMES = ("b2_layernorm", "b2_layernorm_backward_workspace_bytes", "b2_layernorm_backward", "b2_w4_quantize", "b2_w4_dequantize",
         "b2_w4_matvec_workspace_bytes", "b2_w4_matvec")


class Answers:
    """Stands for the extension: every call gives the same answer and is counted."""

    def __init__(self, answer):
        self.answer, self.calls = answer, 0

    def __getattr__(self, name):
        def f(*args):
            self.calls += 1
            return self.answer
        return f


def all_five(t):
    return [lambda: layer.layernorm(4, 8, 1e-5, t, None, None, t), lambda: layer.layernorm_backward(4, 8, t, t, None, t, t, t, None, None),
            lambda: layer.w4_quantize(4, 8, 32, t, t, t), lambda: layer.w4_dequantize(4, 8, 32, t, t, None, t),
            lambda: layer.w4_matvec(4, 8, 8, 32, 1.0, t, t, t, None, 0.0, t)]


@pytest.mark.parametrize("status", [CUDA, TIMEOUT])
def test_an_error_is_raised_and_the_call_not_made_again(built_lib, monkeypatch, status):
    quick = Answers(status)
    monkeypatch.setattr(layer, "_quick", quick)
    monkeypatch.setattr(layer, "_load", lambda: pytest.fail("the call was made a second time"))
    for call in all_five(torch.zeros(4, 8)):
        with pytest.raises(_lib.B2Error) as e:
            call()
        assert e.value.status == status
    assert quick.calls == 5


def test_what_the_extension_does_not_take_goes_to_the_checks(built_lib, monkeypatch):
    quick = Answers(False)
    monkeypatch.setattr(layer, "_quick", quick)
    for call in all_five(torch.zeros(4, 8)):
        with pytest.raises(TypeError, match="expected a CUDA tensor"):
            call()
    assert quick.calls == 5
    monkeypatch.setattr(layer, "_quick", Answers(True))
    t = torch.zeros(4, 8)
    assert layer.layernorm(4, 8, 1e-5, t, None, None, t) is t


@pytest.mark.gpu
@pytest.mark.parametrize("status,raised", [(CUDA, CUDA), (-1, None)])
def test_the_library_is_called_once_and_again_only_after_a_refusal(cuda, status, raised):
    """The extension bound to a stand-in for b2_layernorm that counts its calls and does nothing: after a status that may follow a
    launch the real library is not called, after a refusal (-1) it is."""
    import hpcdeepneuralnetworks_b200 as b2
    b2.default_handle()
    L = layer._load()
    proto = C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_int64, C.c_int64, C.c_float, C.c_int, C.c_void_p, C.c_int64, C.c_int, C.c_void_p, C.c_void_p,
                        C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p)
    calls = []

    def stand_in(*args):
        calls.append(args[1:3])
        return status
    stub = proto(stand_in)
    at = [C.cast(getattr(L, n), C.c_void_p).value for n in NAMES]
    x = torch.randn(5, 64, device="cuda")
    before = x.clone()
    layer._quick.bind(_default, C.cast(stub, C.c_void_p).value, *at[1:])
    try:
        if raised is None:
            layer.layernorm(5, 64, 1e-5, x, None, None, x)
        else:
            with pytest.raises(b2.B2Error) as e:
                layer.layernorm(5, 64, 1e-5, x, None, None, x)
            assert e.value.status == raised
    finally:
        layer._quick.bind(_default, *at)
    assert calls == [(5, 64)]
    once = before.clone()
    layer.layernorm(5, 64, 1e-5, before, None, None, once)
    assert torch.equal(x, once if raised is None else before)


@pytest.mark.gpu
def test_an_error_left_by_an_earlier_call_does_not_touch_these(cuda):
    """The thread's last CUDA error is set (an allocation of 2^60 bytes that the runtime refuses): in-place calls still run once, and
    say so."""
    import hpcdeepneuralnetworks_b200 as b2
    rt = C.CDLL("libcudart.so.12")
    b2.default_handle()
    rows, cols, N = 33, 320, 24
    x, dy = torch.randn(rows, cols, device="cuda"), torch.randn(rows, cols, device="cuda")
    gamma, mean, rstd = torch.rand(cols, device="cuda"), torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    codes, scales, _ = b2.w4_empty(N, cols, 64)

    def everything(x, dy):
        dg = torch.full((cols,), 7.0, device="cuda")
        out = [torch.full((9, N), 7.0, device="cuda"), torch.full((N, cols), 7.0, device="cuda")]
        ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        yield
        b2.layernorm_backward(rows, cols, dy, x, gamma, mean, rstd, dy, dg, None, workspace=ws)
        b2.layernorm(rows, cols, 1e-5, x, gamma, None, x)
        b2.w4_quantize(N, cols, 64, x[:N], codes, scales)
        b2.w4_dequantize(N, cols, 64, codes, scales, None, out[1])
        b2.w4_matvec(9, N, cols, 64, 1.0, x[:9], codes, scales, None, 0.0, out[0], workspace=ws)
        yield [x, dy, dg, codes, scales] + out

    def result(spoil):
        steps = everything(x.clone(), dy.clone())
        next(steps)
        if spoil:
            room = C.c_void_p()
            assert rt.cudaMalloc(C.byref(room), C.c_size_t(1 << 60)) != 0 and rt.cudaPeekAtLastError() != 0
        try:
            got = next(steps)
        finally:
            rt.cudaGetLastError()
        return [t.clone() for t in got]
    for a, b in zip(result(False), result(True)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_an_error_that_a_status_reports_is_not_left_behind(cuda):
    """A runtime call that fails inside the library (the time between two events that were never recorded) comes back as a status;
    the thread's last error, which other code of the process would take for its own, is clear again."""
    import hpcdeepneuralnetworks_b200 as b2
    b2.default_handle()
    L = _lib.load()
    rt = C.CDLL("libcudart.so.12")
    torch.cuda.synchronize()
    timer, ms = C.c_void_p(), C.c_float()
    assert L.b2_timer_create(C.byref(timer)) == 0
    rt.cudaGetLastError()
    assert L.b2_timer_elapsed_ms(timer, C.byref(ms)) == CUDA
    left = rt.cudaGetLastError()
    L.b2_timer_destroy(timer)
    assert left == 0 and b"CUDA error" in L.b2_last_error()


@pytest.mark.parametrize("cols", [8, 8192, 8193, 9000, 100000])
def test_dx_alone_needs_no_workspace(built_lib, cols):
    """As the header says: the workspace may be NULL when neither dgamma nor dbeta is asked for.  Without a device the call gets as far
    as looking for one; a workspace that it wanted would be refused before."""
    if torch.cuda.is_available():
        pytest.skip("there is a device, and these addresses mean nothing to it")
    L = _lib.load()
    at = lambda n: C.c_void_p(n << 30)  # noqa: E731
    call = lambda dg, db, ws, nws: L.b2_layernorm_backward(None, 4, cols, 0, at(1), cols, at(2), cols, 0, at(3), at(4), at(5), at(6), cols, dg, db,  # noqa: E731,E501
                                                           ws, nws, None)
    need = L.b2_layernorm_backward_workspace_bytes(4, cols)
    assert call(None, None, None, 0) == CUDA
    for dg, db in ((at(7), None), (None, at(8)), (at(7), at(8))):
        assert call(dg, db, None, 0) == -6 and call(dg, db, at(9), need - 1) == -6 and call(dg, db, at(9), need) == CUDA


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(4, 9000), (300, 8200), (5, 100001), (3, 4096)])
@pytest.mark.parametrize("inplace", [False, True])
def test_dx_alone_without_a_workspace_equals_dx_beside_the_sums(cuda, rows, cols, inplace):
    import hpcdeepneuralnetworks_b200 as b2
    h = b2.default_handle()
    L = _lib.load()
    x, dy, gamma = torch.randn(rows, cols, device="cuda"), torch.randn(rows, cols, device="cuda"), torch.rand(cols, device="cuda")
    mean, rstd = x.mean(1), x.var(1).rsqrt()
    want, dg, db = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(gamma)
    b2.layernorm_backward(rows, cols, dy, x, gamma, mean, rstd, want, dg, db)
    dx = dy if inplace else torch.full_like(x, 7.0)
    p = [C.c_void_p(t.data_ptr()) for t in (dy, x, gamma, mean, rstd, dx)]
    torch.cuda.synchronize()
    assert L.b2_layernorm_backward(h.raw, rows, cols, 0, p[0], cols, p[1], cols, 0, *p[2:], cols, None, None, None, 0, None) == 0
    torch.cuda.synchronize()
    assert torch.equal(dx, want)
