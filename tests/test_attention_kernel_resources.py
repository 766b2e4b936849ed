"""Register-allocation guard for the kernels of the 8-bit KV cache and of packed prompts, as test_kernel_resources.py
has it for the others: no instantiation touches scratch memory inside a loop. Host-only: compiles to gfx950 assembly."""

from __future__ import annotations

import subprocess
from pathlib import Path

import pytest
from test_kernel_resources import HIPCC, _kernels, _scratch_in_loops

from llmopt.kernels import build


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not available")
@pytest.mark.parametrize("source", ["kvq_write.hip", "kvq_decode.hip", "kvq_chunk.hip", "packed_attention.hip"])
def test_no_spills_in_loops(tmp_path, source):
    src = build.CSRC / "attention" / source
    assert src in build.sources()
    out = tmp_path / (source + ".s")
    flags = [f for f in build.COMPILE_FLAGS if f not in ("-fPIC",)]
    cmd = [HIPCC, *flags, f"-I{build.INCLUDE}", f"-I{build.CSRC}", "--cuda-device-only", "-S", str(src), "-o", str(out)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-2000:]
    kernels = {k: v for k, v in _kernels(out.read_text()).items() if "kernel" in k}
    assert kernels, "no kernels found in the assembly"
    bad = {k: n for k, v in kernels.items() if (n := _scratch_in_loops(v))}
    assert not bad, f"scratch accesses inside loops: {bad}"
