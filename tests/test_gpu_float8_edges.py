"""8-bit floating point at the edges of what its entry points take."""

from __future__ import annotations

import pytest
import torch

from llmopt.kernels import _lib
from llmopt.quantization import float8_linear, quantize_float8
from oracle import float8_oracle as oracle

pytestmark = pytest.mark.gpu

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _bits(t):
    return t.view(torch.uint8)


def _weight(gen, n, k):
    return quantize_float8(torch.randn(n, k, generator=gen, device="cuda") * 0.05, block_rows=128)


def _numbers(t):
    return oracle.numbers(t.codes, t.scales, t.block_rows)


def _stream():
    return torch.cuda.current_stream().cuda_stream


# ---- single rows ------------------------------------------------------------------------------------


@pytest.mark.parametrize("ld", [0, 16, 1008, 5000])
def test_a_single_row_comes_with_any_stride(ld):
    gen, lib = _gen(1), _lib.load_library()
    x, tokens = (quantize_float8(torch.randn(m, 1024, generator=gen, device="cuda")) for m in (1, 2000))
    gate, up, one = _weight(gen, 256, 1024), _weight(gen, 256, 1024), _weight(gen, 1, 1024)
    codes, scales = torch.empty(1, 256, dtype=F8, device="cuda"), torch.empty(1, 2, dtype=E8, device="cuda")
    _lib.call(lib.llmopt_f8_swiglu(x.codes.data_ptr(), ld, x.scales.data_ptr(), 8, 1, 1024, gate.codes.data_ptr(), 1024,
                                   gate.scales.data_ptr(), 8, up.codes.data_ptr(), 1024, up.scales.data_ptr(), 8, 256,
                                   codes.data_ptr(), 256, scales.data_ptr(), 2, None, 0, _stream()), "llmopt_f8_swiglu")
    oracle.check_quantized(codes, scales, *oracle.swiglu(_numbers(x), _numbers(gate), _numbers(up)))
    y = torch.empty(2000, 1, dtype=torch.bfloat16, device="cuda")
    _lib.call(lib.llmopt_f8_linear(tokens.codes.data_ptr(), 1024, tokens.scales.data_ptr(), 8, 2000, 1024, one.codes.data_ptr(), ld,
                                   one.scales.data_ptr(), 8, None, y.data_ptr(), 1, 1, 2, None, 0, _stream()), "llmopt_f8_linear")
    assert torch.equal(y, float8_linear(tokens, one))
