"""What the products in 8-bit floating point hand to their kernels, against a stand-in for the runtime that keeps a launch's
arguments (``hip_arguments_stub.c``). No device is needed."""

from __future__ import annotations

import json
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
LIBRARY = HERE.parent / "quantized-llm-inference-engine-_amd" / "llmopt" / "kernels" / "libllmopt_qlinear.so"

# The library is loaded in a process of its own, behind the stand-in, whose symbols come first there.
CHILD = r"""
import ctypes, json, struct, sys
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
launches, attributes, refuse = (ctypes.c_int.in_dll(stub, "llmopt_stub_" + n) for n in ("launches", "attributes", "refuse"))
block = (ctypes.c_uint * 3).in_dll(stub, "llmopt_stub_block")
argument = (ctypes.c_ubyte * 96).in_dll(stub, "llmopt_stub_argument")
i64, ptr, size = ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t
P = ptr(1 << 20)  # never read: nothing is launched
g = lambda n: i64(-(-n // 128))

def linear(m, n, k, ldx=None, ldw=None):
    return lib.llmopt_f8_linear(P, i64(k if ldx is None else ldx), P, g(k), i64(m), i64(k), P, i64(k if ldw is None else ldw), P,
                                g(k), P, P, i64(n), i64(n), 2, None, size(0), None)

def swiglu(m, n, k, ldx=None, ldg=None, ldu=None):
    return lib.llmopt_f8_swiglu(P, i64(k if ldx is None else ldx), P, g(k), i64(m), i64(k), P, i64(k if ldg is None else ldg), P,
                                g(k), P, i64(k if ldu is None else ldu), P, g(k), i64(n), P, i64(n), P, g(n), None, size(0), None)

def strides():
    word = lambda at: struct.unpack_from("<q", bytes(argument), at)[0]
    return {"x": word(8), "w": word(40), "second": word(72)}

exec(sys.argv[3])
"""


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    cc = shutil.which("cc") or shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    out = tmp_path_factory.mktemp("stub") / "libhip_arguments_stub.so"
    subprocess.run([cc, "-shared", "-fPIC", "-O1", str(HERE / "hip_arguments_stub.c"), "-o", str(out)], check=True)
    return out


def _child(stub, code):
    proc = subprocess.run([sys.executable, "-c", CHILD, str(stub), str(LIBRARY), code], capture_output=True, text=True, timeout=120)
    assert proc.returncode == 0, proc.stderr[-2000:]
    return json.loads(proc.stdout.splitlines()[-1])


@pytest.mark.parametrize("ld", [0, 16, -16, 1008])
@pytest.mark.parametrize("call", ["swiglu(1, 256, 1024, ldx={0})", "linear(2000, 1, 1024, ldw={0})",
                                  "swiglu(2000, 1, 1024, ldg={0}, ldu={0})", "linear(1, 1, 1024, ldx={0}, ldw={0})"])
def test_a_single_rows_stride_is_no_shorter_than_the_row(stub, call, ld):
    """A single row may come with any stride. The tiles take a row's position from it also for the rows behind the last, which
    are to lie behind the operand's end: with a stride below the row's length they would lie in it, and what is read of them
    behind it."""
    got = _child(stub, f"rc = {call.format(ld)}; print(json.dumps([rc, launches.value, strides()]))")
    assert got[0] == 0 and got[1] == 1
    one = {"x"} if "(1, 256" in call else {"x", "w"} if "linear(1" in call else {"w", "second"} if "swiglu" in call else {"w"}
    assert all(got[2][name] == 1024 for name in one), got


@pytest.mark.parametrize("call", ["linear(8192, 4096, 4096)", "linear(1, 4096, 14336)", "swiglu(300, 1280, 2048)"])
def test_the_shared_memory_is_asked_for_with_each_launch(stub, call):
    """The runtime keeps a kernel's shared memory for the device that is current, so a launch on another one asks again, and a failure
    is that call's alone."""
    got = _child(stub, f"""
refuse.value = 1
first = {call}
refuse.value = 0
later = [({call}, attributes.value) for _ in range(3)]
print(json.dumps([first, launches.value, later]))""")
    assert got[0] != 0 and got[1] == 3
    assert got[2] == [[0, 2], [0, 3], [0, 4]]


# The tiles' launch itself, as no entry point calls it. F8TilesArgs: four words of x, four for each weight, then bias, y, ldy, codes, ldc,
# scales, lds, M, N and K, five 32-bit numbers, of which the last two are the parts of K and the steps in each, parts and their stride.
TILES = r"""
launch = lib._ZN6llmopt15launch_f8_tilesERKNS_11F8TilesArgsENS_7F8ShapeEiP12ihipStream_t
def tiles(shape, m, n, k, splits, per, gated=False):
    p = 1 << 20
    weight = [p, k, p, -(-k // 128)]
    block = struct.pack("<22q5i4x2q", p, k, p, -(-k // 128), *weight, *(weight if gated else [0] * 4), 0, p, n, p, n, p, -(-n // 128),
                        m, n, k, 0, 0, 0, splits, per, p, n)
    before = launches.value
    return launch(ctypes.c_char_p(block), shape, 2, None), launches.value - before
"""


def test_the_tiles_refuse_parts_of_k_that_they_have_no_kernel_for(stub):
    """Tiles of 256 tokens and the gated product are whole; a grid of parts would be of tiles that are not there. Neither may a part
    begin behind the last step."""
    code = TILES + "print(json.dumps([tiles(*c) for c in json.loads('''%s''')]))"
    whole = [[shape, 300, 512, 1024, 1, 8] for shape in range(5)]
    parts = [[shape, 300, 512, 1024, 2, 4] for shape in range(1, 5)]
    assert _child(stub, code % json.dumps(whole)) == [[0, 1]] * 5
    assert _child(stub, code % json.dumps(parts)) == [[0, 2]] * 4
    refused = [[0, 300, 512, 1024, 2, 4], [1, 300, 512, 1024, 2, 8], [4, 300, 512, 1024, 8, 2], [0, 300, 512, 1024, 2, 4, True],
               [2, 300, 512, 1024, 2, 4, True], [3, 300, 512, 1024, 1, 8, True]]
    got = _child(stub, code % json.dumps(refused))
    assert all(rc != 0 and launched == 0 for rc, launched in got), got


@pytest.mark.parametrize("tokens", [1, 5, 8, 9, 16])
@pytest.mark.parametrize("n,k", [(128, 1024), (10240, 512), (28672, 2048), (28672, 4096)])
def test_few_tokens_have_waves_by_their_steps(stub, tokens, n, k):
    """A wave takes four steps of 128 columns at a time: up to 16 steps are for four waves at most, 32 for eight."""
    got = _child(stub, f"rc = linear({tokens}, {n}, {k}); print(json.dumps([rc, launches.value, list(block)]))")
    assert got == [0, 1, [256 if k <= 2048 else 512, 1, 1]]
