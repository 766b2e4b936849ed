"""A kernel library or binding built before an entry point was added: what it has still runs, what it lacks says so.
No device is needed."""

from __future__ import annotations

import importlib.machinery
import types

import pytest
import torch

from llmopt.kernels import _lib, ops
from llmopt.quantization import QuantLinear, QuantLinearConfig


class _Older:
    """The built library without the entry points whose names contain ``lacks``."""

    def __init__(self, real, lacks, version=None):
        self.__dict__.update(_real=real, _lacks=lacks, _version=version)

    def __getattr__(self, name):
        if self._lacks in name:
            raise AttributeError(f"undefined symbol: {name}")
        if name == "llmopt_q_abi_version" and self._version is not None:
            return lambda: self._version
        return getattr(self._real, name)


@pytest.fixture
def fresh(monkeypatch):
    real = _lib.load_library()
    for name, value in (("_handle", None), ("_binding", None), ("_binding_tried", False)):
        monkeypatch.setattr(_lib, name, value)
    return monkeypatch, real


def _no_native_path():
    module = QuantLinear(128, 64, QuantLinearConfig(4, 128, True, torch.bfloat16), bias=False)
    with pytest.warns(RuntimeWarning, match="native host path"):
        assert ops.module_linear(torch.zeros(1, 128, dtype=torch.bfloat16), module, 64) is None


def test_a_library_without_the_cache_entry_points(fresh):
    patch, real = fresh
    patch.setattr(_lib.ctypes, "CDLL", lambda path: _Older(real, "kvq"))
    lib = _lib.load_library()
    assert lib.llmopt_q_linear_workspace(1, 4096, 4096, 4, 128) == 0
    with pytest.raises(RuntimeError, match="llmopt_kvq_write.*[Bb]uild it again"):
        lib.llmopt_kvq_write()
    _no_native_path()


def test_another_abi_version_is_named_before_missing_entry_points(fresh):
    patch, real = fresh
    patch.setattr(_lib.ctypes, "CDLL", lambda path: _Older(real, "kvq", version=0))
    with pytest.raises(RuntimeError, match="ABI version 0"):
        _lib.load_library()


def test_a_binding_without_the_cache_entry_points(fresh):
    patch, _ = fresh

    def older(self, module):
        module.torch_version = torch.__version__.split("+")[0]
        module.attach = lambda *addresses: None

    patch.setattr(importlib.machinery.ExtensionFileLoader, "create_module", lambda self, spec: types.ModuleType(spec.name))
    patch.setattr(importlib.machinery.ExtensionFileLoader, "exec_module", older)
    _no_native_path()
