"""8-bit floating point without columns, tokens or features, on the host. No device is needed."""

from __future__ import annotations

import pytest
import torch

from llmopt.quantization import float8_linear, float8_swiglu, quantize_float8, rmsnorm_float8


@pytest.mark.parametrize("lead", [(), (3,), (0,), (2, 3), (2, 0)])
def test_no_columns(lead):
    x, w = quantize_float8(torch.zeros(*lead, 0)), quantize_float8(torch.zeros(5, 0), block_rows=128)
    assert x.codes.shape == x.scales.shape == (*lead, 0) and w.scales.shape == (1, 0)
    assert x.dequantize().shape == (*lead, 0)
    bias = torch.arange(5, dtype=torch.bfloat16)
    assert torch.equal(float8_linear(x, w, bias), bias.expand(*lead, 5))
    act = float8_swiglu(x, w, w)
    assert act.codes.shape == (*lead, 5) and act.scales.shape == (*lead, 1) and not bool(act.dequantize().any())
    out, h = rmsnorm_float8(torch.zeros(*lead, 0), torch.zeros(0), 1e-5, residual=torch.zeros(*lead, 0))
    assert out.codes.shape == h.shape == (*lead, 0)


@pytest.mark.parametrize("lead", [(0,), (2, 0)])
def test_no_tokens(lead):
    x, w = quantize_float8(torch.zeros(*lead, 200)), quantize_float8(torch.ones(5, 200), block_rows=128)
    assert x.scales.shape == (*lead, 2)
    assert float8_linear(x, w).shape == (*lead, 5) and float8_swiglu(x, w, w).codes.shape == (*lead, 5)


def test_no_features():
    x, w = quantize_float8(torch.ones(3, 200)), quantize_float8(torch.zeros(0, 200), block_rows=128)
    assert w.scales.shape == (0, 2)
    assert float8_linear(x, w).shape == (3, 0) and float8_swiglu(x, w, w).scales.shape == (3, 0)
