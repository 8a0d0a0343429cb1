"""CPU tests of how the extension of the layer operators' calls is built and taken: anew for another torch, not at all without one,
and never where it was made for a torch that is not the one running."""
import importlib
import os
import types

import pytest
import torch

from hpcdeepneuralnetworks_b200 import build, layer


@pytest.fixture
def compiler(built_lib, monkeypatch, tmp_path):
    """Paths of its own, and a compiler that writes an empty file and is counted."""
    monkeypatch.setattr(build, "CALLS", str(tmp_path / "_calls.so"))
    monkeypatch.setattr(build, "CALLS_STAMP", str(tmp_path / "calls.stamp"))
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        open(build.CALLS, "w").close()
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")
    monkeypatch.setattr(build.subprocess, "run", run)
    return calls


def test_built_once_and_again_for_another_torch_or_when_forced(compiler, monkeypatch):
    found = build._torch()
    assert found is not None and found[1] == torch.__version__ and os.path.samefile(found[0], os.path.dirname(torch.__file__))
    for _ in range(2):
        assert build.build_calls() == build.CALLS
        assert len(compiler) == 1
    build.build_calls(force=True)
    assert len(compiler) == 2
    monkeypatch.setattr(build, "_torch", lambda: (found[0], "99.0+cu999"))
    build.build_calls()
    assert len(compiler) == 3 and any("99.0+cu999" in a for a in compiler[-1])
    build.build_calls()
    assert len(compiler) == 3
    os.remove(build.CALLS_STAMP)
    build.build_calls()
    assert len(compiler) == 4


def test_forced_builds_reach_the_extension(built_lib, monkeypatch):
    seen = []
    monkeypatch.setattr(build, "build_calls", lambda force=False: seen.append(force))
    build.build()
    assert seen == [False]
    monkeypatch.setattr(build, "build_driver", lambda: None)
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: types.SimpleNamespace(returncode=0, stdout="", stderr=""))
    build.build(force=True)
    assert seen == [False, True]


@pytest.mark.parametrize("what", ["no torch", "a torch without CUDA", "no Python.h"])
def test_the_library_is_built_without_a_torch_for_cuda(compiler, monkeypatch, tmp_path, what):
    if what == "no Python.h":
        monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    else:
        spec = None if what == "no torch" else types.SimpleNamespace(submodule_search_locations=[str(tmp_path)])
        monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: spec)
        assert build._torch() is None
    assert build.build_calls() is None and build.build_calls(force=True) is None
    assert not compiler


@pytest.mark.parametrize("module", [None, types.SimpleNamespace(torch_version="0.1"), types.SimpleNamespace()])
def test_calls_go_through_the_checks_without_it(built_lib, monkeypatch, module):
    def find(name):
        if module is None:
            raise ImportError("undefined symbol")
        return module
    monkeypatch.setattr(layer, "_quick", None)
    monkeypatch.setattr(layer, "_looked", False)
    monkeypatch.setattr(importlib, "import_module", find)
    with pytest.warns(RuntimeWarning, match="hpcdeepneuralnetworks_b200.build"):
        assert layer._load() is layer._lib.load()
    assert layer._quick is None
    assert layer._load() is layer._lib.load()          # said once
    assert layer.layernorm_backward_workspace_bytes(4, 8) > 0
    t = torch.zeros(4, 8)
    with pytest.raises(TypeError, match="expected a CUDA tensor"):
        layer.layernorm(4, 8, 1e-5, t, None, None, t)


def test_the_extension_that_was_built_is_taken(built_lib):
    layer._load()
    assert layer._quick is not None and layer._quick.torch_version == torch.__version__


def test_an_operator_replaced_in_its_module_is_seen_in_the_package(built_lib, monkeypatch):
    import hpcdeepneuralnetworks_b200 as b2
    for module, name in ((b2.blas, "sgemm"), (layer, "layernorm")):
        real = getattr(b2, name)
        assert real is getattr(module, name)
        with monkeypatch.context() as m:
            m.setattr(module, name, lambda *a: "replaced")
            assert getattr(b2, name)() == "replaced"
        assert getattr(b2, name) is real
        with monkeypatch.context() as m:          # or in the package itself, there alone
            m.setattr(b2, name, lambda *a: "here")
            assert getattr(b2, name)() == "here" and getattr(module, name) is real
        assert getattr(b2, name) is real
    with pytest.raises(AttributeError):
        b2.no_such_operator
