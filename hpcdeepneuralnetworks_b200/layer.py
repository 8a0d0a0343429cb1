"""Operators of a layer around the matrix products, over the same C ABI: layer norm with its gradients, and 4-bit weights
with group scales (quantise, expand, matrix-vector product).

The conventions are those of ``blas``: sizes first, torch CUDA tensors as device memory, work enqueued on the current
stream, outputs given by the caller and returned, errors as ``B2Error``.  Tensors may be float32, bfloat16 or float16 and
must lie on the current device.  A matrix is a 2-D tensor whose rows are contiguous (a column slice of a wider one
included: its row stride is the leading dimension), or a contiguous tensor of any shape with enough elements; a leading
dimension given by name (in elements; ``ldq`` in bytes) takes the tensor as raw memory of that pitch.
"""
from __future__ import annotations

import ctypes
import functools
import importlib
import warnings

import torch

from . import _lib
from ._lib import check
from .blas import Handle, _default, default_handle

TYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
W4_GROUPS = (32, 64, 128, 256)
W4_MAX_ROWS = 64

# csrc/calls.cpp: the usual calls, checked and made without the Python below (which decides all others, with the same results)
_quick = None
_looked = False


def _load():
    """The library; the first call hands its functions to ``_calls``.  Where that is missing, or was built for another torch, whose
    tensors it would misread, every call goes through the checks below: slower, with the same results."""
    global _quick, _looked
    L = _lib.load()
    if not _looked:
        _looked = True
        try:
            quick = importlib.import_module(__package__ + "._calls")
            why = None if quick.torch_version == torch.__version__ else f"was built for torch {quick.torch_version}, this is {torch.__version__}"
        except (ImportError, AttributeError) as e:
            why = f"cannot be used ({e})"
        if why:
            warnings.warn(f"_calls.so {why}: calls of the layer operators take some microseconds longer; "
                          "`python -m hpcdeepneuralnetworks_b200.build` makes it again", RuntimeWarning, stacklevel=3)
        else:
            names = ("b2_layernorm", "b2_layernorm_backward_workspace_bytes", "b2_layernorm_backward", "b2_w4_quantize", "b2_w4_dequantize",
                     "b2_w4_matvec_workspace_bytes", "b2_w4_matvec")
            quick.bind(_default, *(ctypes.cast(getattr(L, n), ctypes.c_void_p).value for n in names))
            _quick = quick
    return L


def _done(answer) -> bool:
    """Whether the extension made the call.  A status that may have come after a launch is an error, never a reason to call again."""
    return answer is True or (answer is not False and check(answer) >= 0)


_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _stream(device: int) -> int:
    # the current stream's handle without building a Stream object (about a microsecond of a small call)
    return _raw_stream(device) if _raw_stream else torch.cuda.current_stream(device).cuda_stream


def _tensor(t, name, device=None):
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise TypeError(f"{name}: expected a CUDA tensor")
    if device is not None and t.get_device() != device:
        raise ValueError(f"{name} lies on device {t.get_device()}, but device {device} is current")
    return t


def _type(t, name) -> int:
    code = TYPE_CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name}: {t.dtype} is not float32, bfloat16 or float16")
    return code


def _same_type(t, dtype, name):
    if t.dtype is not dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")


def _matrix(t, rows, cols, ld, name, device):
    """(address, leading dimension) of a rows x cols matrix held by ``t``."""
    if ld is None and isinstance(t, torch.Tensor) and t.get_device() == device and t.shape == (rows, cols) and t.is_contiguous():
        return t.data_ptr(), cols      # the usual case, first
    _tensor(t, name, device)
    if ld is None:
        if t.dim() > 1 and t.shape[-1] != cols:
            raise ValueError(f"{name}: rows of shape {tuple(t.shape)} are not {cols} long (a pitch is given by name)")
        if t.is_contiguous():
            if t.numel() < rows * cols:
                raise ValueError(f"{name}: {t.numel()} elements are too few for {rows} x {cols}")
            return t.data_ptr(), cols
        if t.dim() != 2 or t.shape[0] < rows or (cols > 1 and t.stride(1) != 1):
            raise ValueError(f"{name}: neither contiguous nor a {rows} x {cols} matrix with contiguous rows")
        return t.data_ptr(), t.stride(0) if rows > 1 else cols
    if rows > 0 and cols > 0:
        held = t.untyped_storage().nbytes() // t.element_size() - t.storage_offset()
        if ld >= cols and held < (rows - 1) * ld + cols:
            raise ValueError(f"{name}: {held} elements are too few for {rows} rows of {cols} that lie {ld} apart")
    return t.data_ptr(), ld


def _vector(t, n, name, device, dtype=None):
    """Address of a contiguous vector of at least n elements, or None."""
    if t is None:
        return None
    if isinstance(t, torch.Tensor) and t.get_device() == device and t.is_contiguous() and t.numel() >= n and (dtype is None or t.dtype is dtype):
        return t.data_ptr()            # the usual case, first
    _tensor(t, name, device)
    if dtype is not None:
        _same_type(t, dtype, name)
    if not t.is_contiguous() or t.numel() < n:
        raise ValueError(f"{name}: expected {n} contiguous elements, got shape {tuple(t.shape)}, strides {t.stride()}")
    return t.data_ptr()


def _params_type(x, params, names):
    """The common element type of the layer norm's parameter tensors that are given: float32 or x's."""
    dtype = None
    for t, name in zip(params, names):
        if t is None or (dtype is not None and isinstance(t, torch.Tensor) and t.dtype is dtype):
            continue
        _tensor(t, name)
        if t.dtype is not torch.float32 and t.dtype is not x.dtype:
            raise TypeError(f"{name}: {t.dtype} is neither float32 nor x's {x.dtype}")
        if dtype is not None:
            raise TypeError(f"{name}: {t.dtype} differs from the other parameters' {dtype}")
        dtype = t.dtype
    return TYPE_CODES[dtype if dtype is not None else x.dtype]


def _raw(handle, device):
    """The library's handle: the caller's, or the default one of the device."""
    h = handle or _default.get(device) or default_handle()
    return h.raw


# ---- layer norm ---------------------------------------------------------------------------------
def layernorm(rows, cols, eps, x, gamma, beta, y=None, *, mean=None, rstd=None, ldx=None, ldy=None, handle: Handle | None = None):
    """y = (x - mean) * rstd * gamma + beta over the rows of x.  ``gamma``, ``beta``: ``cols`` elements of float32 or x's
    type, or None.  ``mean``, ``rstd``: float32 tensors of ``rows`` elements that receive the statistics, or None.
    ``y``: x's type, x itself for the norm in place, or None for a new tensor.  Returns ``y``."""
    if _quick and ldx is None and ldy is None and _done(_quick.layernorm(handle, rows, cols, eps, x, gamma, beta, y, mean, rstd)):
        return y
    _tensor(x, "x")
    device = torch.cuda.current_device()
    if y is None:
        y = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
    t = _type(x, "x")
    px, ldx = _matrix(x, rows, cols, ldx, "x", device)
    py, ldy = _matrix(y, rows, cols, ldy, "y", device)
    _same_type(y, x.dtype, "y")
    pt = _params_type(x, (gamma, beta), ("gamma", "beta"))
    check(_load().b2_layernorm(_raw(handle, device), rows, cols, eps, t, px, ldx, pt, _vector(gamma, cols, "gamma", device),
                                   _vector(beta, cols, "beta", device), py, ldy, _vector(mean, rows, "mean", device, torch.float32),
                                   _vector(rstd, rows, "rstd", device, torch.float32), _stream(device)))
    return y


@functools.lru_cache(maxsize=4096)
def _layernorm_workspace(rows, cols) -> int:
    return int(_load().b2_layernorm_backward_workspace_bytes(rows, cols))


def layernorm_backward_workspace_bytes(rows: int, cols: int) -> int:
    """Bytes that the sums of ``layernorm_backward`` go through."""
    return _layernorm_workspace(rows, cols)


def layernorm_backward(rows, cols, dy, x, gamma, mean, rstd, dx, dgamma, dbeta, *, lddy=None, ldx=None, lddx=None,
                       workspace=None, handle: Handle | None = None):
    """Gradients of ``layernorm`` from dy and the forward pass's ``mean`` and ``rstd``; ``dx`` (x's type), ``dgamma`` and
    ``dbeta`` (gamma's type) are each written unless None.  ``workspace``: a tensor of at least
    ``layernorm_backward_workspace_bytes(rows, cols)`` bytes that no other call uses meanwhile; None takes one from torch's
    allocator on the current stream for this call.  Returns ``(dx, dgamma, dbeta)``."""
    if _quick and lddy is None and ldx is None and lddx is None and \
            _done(_quick.layernorm_backward(handle, rows, cols, dy, x, gamma, mean, rstd, dx, dgamma, dbeta, workspace)):
        return dx, dgamma, dbeta
    L = _load()
    _tensor(x, "x")
    device = torch.cuda.current_device()
    t = _type(x, "x")
    px, ldx = _matrix(x, rows, cols, ldx, "x", device)
    pdy, lddy = _matrix(dy, rows, cols, lddy, "dy", device)
    _same_type(dy, x.dtype, "dy")
    pdx, lddx = (None, cols) if dx is None else _matrix(dx, rows, cols, lddx, "dx", device)
    if dx is not None:
        _same_type(dx, x.dtype, "dx")
    pt = _params_type(x, (gamma, dgamma, dbeta), ("gamma", "dgamma", "dbeta"))
    ws, ws_bytes = None, 0
    if workspace is not None:
        ws, ws_bytes = _vector(workspace, 0, "workspace", device), workspace.numel() * workspace.element_size()
    elif rows > 0 and (dgamma is not None or dbeta is not None):
        ws_bytes = _layernorm_workspace(rows, cols)
        workspace = x.new_empty(-(-ws_bytes // x.element_size()))
        ws = workspace.data_ptr()
    check(L.b2_layernorm_backward(_raw(handle, device), rows, cols, t, pdy, lddy, px, ldx, pt, _vector(gamma, cols, "gamma", device),
                                  _vector(mean, rows, "mean", device, torch.float32), _vector(rstd, rows, "rstd", device, torch.float32),
                                  pdx, lddx, _vector(dgamma, cols, "dgamma", device), _vector(dbeta, cols, "dbeta", device),
                                  ws, ws_bytes, _stream(device)))
    return dx, dgamma, dbeta


# ---- 4-bit weights ----------------------------------------------------------------------------
def w4_empty(N, K, group, scale_dtype=torch.bfloat16, zeros=False):
    """Tensors for the 4-bit form of an N x K matrix on the current device: ``(codes, scales, zeros)``.  ``codes`` is an
    N x ceil(K/2) view of rows that start on 16-byte boundaries, as the products read them fastest."""
    if group not in W4_GROUPS:
        raise ValueError(f"group {group} is not one of {W4_GROUPS}")
    if scale_dtype not in TYPE_CODES:
        raise TypeError(f"scales of {scale_dtype} are not float32, bfloat16 or float16")
    width, groups = (K + 1) // 2, -(-K // group)
    codes = torch.empty((N, -(-width // 16) * 16), dtype=torch.uint8, device="cuda")[:, :width]
    scales = torch.empty((N, groups), dtype=scale_dtype, device="cuda")
    return codes, scales, torch.empty((N, groups), dtype=torch.uint8, device="cuda") if zeros else None


def _w4(N, K, group, codes, scales, zeros, ldq, device):
    """The arguments (codes, ldq, scale type, scales, zeros) that the calls on 4-bit weights share."""
    if group not in W4_GROUPS:
        raise ValueError(f"group {group} is not one of {W4_GROUPS}")
    pq, ldq = _matrix(codes, N, (K + 1) // 2, ldq, "codes", device)
    _same_type(codes, torch.uint8, "codes")
    count = N * -(-K // group)
    ps = _vector(scales, count, "scales", device)
    if ps is None:
        raise TypeError("scales: expected a CUDA tensor")
    return pq, ldq, _type(scales, "scales"), ps, _vector(zeros, count, "zeros", device, torch.uint8)


def w4_quantize(N, K, group, W, codes, scales, zeros=None, *, ldw=None, ldq=None, handle: Handle | None = None):
    """Quantises W (N x K) to 4 bits in groups of ``group`` along K: ``codes`` (uint8, two per byte), ``scales`` (any of the
    three types) and, when ``zeros`` (uint8) is given, zero points; otherwise symmetric around 8.  ``w4_empty`` makes the
    three tensors.  Returns ``(codes, scales, zeros)``."""
    if _quick and ldw is None and ldq is None and _done(_quick.w4_quantize(handle, N, K, group, W, codes, scales, zeros)):
        return codes, scales, zeros
    _tensor(W, "W")
    device = torch.cuda.current_device()
    t = _type(W, "W")
    pw, ldw = _matrix(W, N, K, ldw, "W", device)
    pq, ldq, st, ps, pz = _w4(N, K, group, codes, scales, zeros, ldq, device)
    check(_load().b2_w4_quantize(_raw(handle, device), N, K, group, t, pw, ldw, pq, ldq, st, ps, pz, _stream(device)))
    return codes, scales, zeros


def w4_dequantize(N, K, group, codes, scales, zeros=None, W=None, *, transpose=False, dtype=torch.float32, ldw=None, ldq=None,
                  handle: Handle | None = None):
    """Expands 4-bit weights to ``W``: N x K, or K x N with ``transpose`` (then the right operand of
    ``sgemm(M, N, K, alpha, X, W, beta, C)`` for C = X * W^T).  ``W`` None: a new tensor of ``dtype``.  Returns ``W``."""
    if _quick and ldw is None and ldq is None and \
            _done(_quick.w4_dequantize(handle, N, K, group, codes, scales, zeros, 1 if transpose else 0, W)):
        return W
    _tensor(codes, "codes")
    device = torch.cuda.current_device()
    rows, cols = (K, N) if transpose else (N, K)
    if W is None:
        W = torch.empty((rows, cols), dtype=dtype, device=codes.device)
    pw, ldw = _matrix(W, rows, cols, ldw, "W", device)
    pq, ldq, st, ps, pz = _w4(N, K, group, codes, scales, zeros, ldq, device)
    check(_load().b2_w4_dequantize(_raw(handle, device), N, K, group, pq, ldq, st, ps, pz, _type(W, "W"), pw, ldw, 1 if transpose else 0,
                                       _stream(device)))
    return W


@functools.lru_cache(maxsize=4096)
def _w4_matvec_workspace(M, N, K, t) -> int:
    return int(_load().b2_w4_matvec_workspace_bytes(M, N, K, t))


def w4_matvec_workspace_bytes(M: int, N: int, K: int, dtype) -> int:
    """Bytes that ``w4_matvec`` lays x out in; 0 for smaller products."""
    return _w4_matvec_workspace(M, N, K, TYPE_CODES[dtype])


def w4_matvec(M, N, K, group, alpha, x, codes, scales, zeros, beta, y=None, *, ldx=None, ldy=None, ldq=None,
              workspace=None, handle: Handle | None = None):
    """y = alpha * x * W^T + beta * y with W (N x K) in 4-bit form, x (M x K) and y (M x N) of one type, M = 0..64 rows (more:
    ``w4_dequantize`` once and ``sgemm``).  ``y`` None: a new tensor (beta must be 0).  ``workspace``: a tensor of at least
    ``w4_matvec_workspace_bytes(M, N, K, x.dtype)`` bytes that no other call uses meanwhile; None takes one from torch's allocator
    on the current stream for this call.  Returns ``y``."""
    if _quick and ldx is None and ldy is None and ldq is None and \
            _done(_quick.w4_matvec(handle, M, N, K, group, alpha, x, codes, scales, zeros, beta, y, workspace)):
        return y
    _tensor(x, "x")
    device = torch.cuda.current_device()
    if y is None:
        if beta != 0:
            raise ValueError("beta is not 0, but there is no y to read")
        y = torch.empty((M, N), dtype=x.dtype, device=x.device)
    t = _type(x, "x")
    px, ldx = _matrix(x, M, K, ldx, "x", device)
    py, ldy = _matrix(y, M, N, ldy, "y", device)
    _same_type(y, x.dtype, "y")
    pq, ldq, st, ps, pz = _w4(N, K, group, codes, scales, zeros, ldq, device)
    ws, ws_bytes = None, 0
    if workspace is None:
        ws_bytes = _w4_matvec_workspace(M, N, K, t)
        if ws_bytes:
            workspace = x.new_empty(ws_bytes // x.element_size())      # a multiple of 16 bytes
            ws = workspace.data_ptr()
    else:
        ws, ws_bytes = _vector(workspace, 0, "workspace", device), workspace.numel() * workspace.element_size()
    check(_load().b2_w4_matvec(_raw(handle, device), M, N, K, group, alpha, t, px, ldx, pq, ldq, st, ps, pz, beta, py, ldy, ws, ws_bytes, _stream(device)))
    return y
