"""Of the entry points in 8-bit floating point, a call any of whose kernels fails to launch reports it (against the stand-in of
``hip_launch_stub.c``, each launch failing in turn), and how many launches each path makes. And a kernel library or binding built
before them serves the others. No device is needed."""

from __future__ import annotations

import ctypes
import importlib.machinery
import json
import shutil
import subprocess
import sys
import types
from pathlib import Path

import pytest
import torch

from llmopt.kernels import _lib, float8_ops
from llmopt.quantization import quantize_float8

HERE = Path(__file__).resolve().parent
LIBRARY = HERE.parent / "quantized-llm-inference-engine-_amd" / "llmopt" / "kernels" / "libllmopt_qlinear.so"

# The library is loaded in a process of its own, behind the stand-in, whose symbols come first there.
CHILD = r"""
import ctypes, json, sys
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
launches, fail = (ctypes.c_int.in_dll(stub, "llmopt_stub_" + n) for n in ("launches", "fail"))
i64, ptr, f32, size = ctypes.c_int64, ctypes.c_void_p, ctypes.c_float, ctypes.c_size_t
for name in ("llmopt_f8_linear_workspace", "llmopt_f8_swiglu_workspace"):
    getattr(lib, name).restype = size
P = ptr(1 << 20)  # never read: nothing is launched
g = lambda n: i64(-(-n // 128))

def quantize(rows, cols, block, dtype=2):
    return lib.llmopt_f8_quantize(P, i64(cols), dtype, i64(rows), i64(cols), i64(block), P, i64(cols), P, g(cols), None)

def norm(rows, hidden, residual):
    return lib.llmopt_f8_rmsnorm(P, i64(hidden), P if residual else None, i64(hidden), P, i64(hidden), P, P, i64(hidden), P, g(hidden),
                                 i64(rows), i64(hidden), f32(1e-5), 2, None)

def linear(m, n, k, short=False):
    need = 0 if short else lib.llmopt_f8_linear_workspace(i64(m), i64(n), i64(k))
    return lib.llmopt_f8_linear(P, i64(k), P, g(k), i64(m), i64(k), P, i64(k), P, g(k), P, P, i64(n), i64(n), 2,
                                P if need else None, size(need), None)

def swiglu(m, n, k, short=False):
    need = 0 if short else lib.llmopt_f8_swiglu_workspace(i64(m), i64(n), i64(k))
    return lib.llmopt_f8_swiglu(P, i64(k), P, g(k), i64(m), i64(k), P, i64(k), P, g(k), P, i64(k), P, g(k), i64(n), P, i64(n), P,
                                g(n), P if need else None, size(need), None)

case = json.loads(sys.argv[3])
call = lambda: globals()[case[0]](*case[1])
rc = call()
total = launches.value
got = []
for at in range(1, total + 1):
    launches.value, fail.value = 0, at
    got.append(call())
fail.value = 0
print(json.dumps({"rc": rc, "launches": total, "failed": got, "after": call()}))
"""

CASES = {  # name: (call, arguments, launches)
    "rows quantized": ("quantize", [5, 100, 1], 1),
    "a weight quantized": ("quantize", [300, 1000, 128, 0], 1),
    "more rows quantized than a launch counts": ("quantize", [1 << 24, 100, 1], 2),
    "and in several workgroups a row": ("quantize", [1 << 23, 5000, 1, 1], 2),
    "norm": ("norm", [5, 4096, True], 1),
    "norm of long rows": ("norm", [5, 9000, False], 1),
    "more rows normed than a launch counts": ("norm", [1 << 24, 64, True], 2),
    "one token": ("linear", [1, 4096, 4096], 1),
    "few tokens": ("linear", [40, 1536, 1024], 1),
    "parts of K and their join": ("linear", [32, 4096, 14336], 2),
    "without the workspace": ("linear", [32, 4096, 14336, True], 1),
    "tiles": ("linear", [8192, 4096, 14336], 1),
    "any rows": ("linear", [33, 50, 77], 1),
    "the gated product of few tokens": ("swiglu", [4, 14336, 4096], 2),
    "and without the workspace": ("swiglu", [4, 14336, 4096, True], 1),
    "gated tiles": ("swiglu", [1000, 14336, 4096], 1),
    "gated, any rows": ("swiglu", [33, 50, 77], 1),
    "no tokens": ("linear", [0, 4096, 4096], 0),
}


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    cc = shutil.which("cc") or shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    out = tmp_path_factory.mktemp("stub") / "libhip_launch_stub.so"
    subprocess.run([cc, "-shared", "-fPIC", "-O1", str(HERE / "hip_launch_stub.c"), "-o", str(out)], check=True)
    return out


@pytest.mark.parametrize("name", CASES)
def test_a_failed_launch_is_reported(stub, name):
    call, args, launches = CASES[name]
    proc = subprocess.run([sys.executable, "-c", CHILD, str(stub), str(LIBRARY), json.dumps([call, args])],
                          capture_output=True, text=True, timeout=120)
    assert proc.returncode == 0, proc.stderr[-2000:]
    got = json.loads(proc.stdout.splitlines()[-1])
    assert got["rc"] == 0 and got["launches"] == launches and got["after"] == 0
    assert all(rc != 0 for rc in got["failed"]), got


def test_unaligned_products_of_more_workgroups_than_a_launch_counts_are_refused():
    lib, p = _lib.load_library(), 1 << 20
    rows = 1 << 23
    assert lib.llmopt_f8_linear(p, 77, p, 1, rows, 77, p, 77, p, 1, None, p, 4096, 4096, 2, None, 0, None) == -2
    assert b"workgroups" in lib.llmopt_f8_last_error()
    assert lib.llmopt_f8_swiglu(p, 77, p, 1, rows, 77, p, 77, p, 1, p, 77, p, 1, 4096, p, 4096, p, 32, None, 0, None) == -2
    assert b"workgroups" in lib.llmopt_f8_last_error()


# ---- older builds -----------------------------------------------------------------------------------


class _Older:
    """The built library without the entry points of 8-bit floating point."""

    def __init__(self, real):
        self.__dict__["_real"] = real

    def __getattr__(self, name):
        if "_f8_" in name:
            raise AttributeError(f"undefined symbol: {name}")
        return getattr(self._real, name)


@pytest.fixture
def fresh(monkeypatch):
    real = _lib.load_library()
    for name, value in (("_handle", None), ("_binding", None), ("_binding_tried", False)):
        monkeypatch.setattr(_lib, name, value)
    return monkeypatch, real


def test_a_library_from_before_them(fresh):
    patch, real = fresh
    patch.setattr(ctypes, "CDLL", lambda path: _Older(real))
    lib = _lib.load_library()
    assert lib.llmopt_q_linear_workspace(1, 4096, 4096, 4, 128) == 0
    with pytest.raises(RuntimeError, match="llmopt_f8_linear.*[Bb]uild it again"):
        lib.llmopt_f8_linear()
    with pytest.warns(RuntimeWarning, match="native host path"):
        assert float8_ops.native().f8_quantize(torch.zeros(1, 8), 1) is None
    assert quantize_float8(torch.ones(1, 8)).scales.float().item() == 2.0**-8  # the host needs none of it: 1 <= 448 / 2^8


def test_a_binding_from_before_them(fresh):
    patch, _ = fresh

    def older(self, module):
        module.torch_version = torch.__version__.split("+")[0]
        module.attach = lambda *addresses: None
        module.attach_kvq = lambda *addresses: None

    patch.setattr(importlib.machinery.ExtensionFileLoader, "create_module", lambda self, spec: types.ModuleType(spec.name))
    patch.setattr(importlib.machinery.ExtensionFileLoader, "exec_module", older)
    with pytest.warns(RuntimeWarning, match="native host path.*attach_f8"):
        float8_ops.native()
    for name in ("f8_check", "f8_quantize", "f8_rmsnorm", "f8_linear", "f8_swiglu"):
        assert getattr(float8_ops.native(), name)() is None
