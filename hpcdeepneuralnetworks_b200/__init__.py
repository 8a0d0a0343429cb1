"""B200-native (sm_100a) FP32 BLAS-kernel library: row-major SGEMM (FFMA and 3xTF32 paths),
ABFT fault-tolerant SGEMM, SAXPY and SDOT behind the reference project's launcher signatures, and
the operators of a layer around those products: layer norm with its gradients, and matrix-vector
products with 4-bit weights.

The arithmetic lives in ``libb2blas.so`` (hand-written CUDA, C ABI in ``include/b2blas.h``);
this package is the host-side mirror of the reference interface and uses PyTorch only for
device memory, streams and ``torch.distributed``.
"""
from ._lib import B2Error, Fault, FtReport, LIB_PATH  # noqa: F401


import sys as _sys
import types as _types


class _Live:
    """An operator of this package that has been asked for: looked up in its module each time, so that what is replaced there is seen
    here (0.1 us an access; through ``__getattr__`` each time 0.5)."""

    def __init__(self, module, name):
        self.module, self.name = module, name

    def __get__(self, package, kind):
        return getattr(self.module, self.name)


class _Package(_types.ModuleType):
    pass


_sys.modules[__name__].__class__ = _Package


def __getattr__(name):
    # Operators are resolved lazily so that importing the package (and building the library)
    # works on a machine without a GPU; using an operator without the built library raises.
    import importlib
    if name in ("blas", "build", "dist", "gen_ft_sgemm", "layer", "_lib"):
        return importlib.import_module(f"{__name__}.{name}")
    for module in ("blas", "layer"):
        m = importlib.import_module(f"{__name__}.{module}")
        if hasattr(m, name):
            setattr(_Package, name, _Live(m, name))
            return getattr(m, name)
    raise AttributeError(name)
