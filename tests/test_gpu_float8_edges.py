"""8-bit floating point at the edges of what its entry points take."""

from __future__ import annotations

import pytest
import torch

from llmopt.kernels import _lib
from llmopt.quantization import Float8Tensor, float8_linear, float8_swiglu, quantize_float8
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


# ---- maxima next to a border of the scales -----------------------------------------------------------


def _strong(gen, m, k, share, gain):
    """Rows in which a share of the channels is `gain` times as strong as the rest."""
    return torch.randn(m, k, generator=gen, device="cuda") * torch.where(torch.rand(k, generator=gen, device="cuda") < share, gain, 1.0)


def _exact_scales(x, gate, up, n):
    """The least and the greatest exponent of each group's scale for sums that are off by 1e-5: fp32 sums of a few thousand products of
    either sign are off by a few 2^-24 of their terms' typical size, and the largest of 128 of them is no sum that its terms cancel in."""
    want, _ = oracle.swiglu(_numbers(x), _numbers(gate), _numbers(up))
    amax = want.abs().view(-1, n // 128, 128).amax(2)
    return [torch.ceil(torch.log2(amax * (1 + off) / 448.0)) for off in (-1e-5, 1e-5)]


@pytest.mark.parametrize("share,gain", [(0.01, 8.0), (0.005, 30.0), (0.002, 100.0), (0.001, 1000.0)])
@pytest.mark.parametrize("at_once,k", [(16, 1024), (512, 1024), (1024, 2048)])
def test_scales_are_those_of_exact_sums_where_a_few_channels_are_strong(at_once, k, share, gain):
    """A strong channel's product takes bits of the seven beside it: sums are off by 1e-4 of the largest and more, many times what they
    are for channels of like strength."""
    gen, m, n = _gen(31), 4096, 14336
    gate, up = _weight(gen, n, k), _weight(gen, n, k)
    x = quantize_float8(_strong(gen, m, k, share, gain))
    for first in range(0, m, at_once if at_once > 16 else 1024):
        rows = slice(first, first + at_once)
        part = Float8Tensor(x.codes[rows], x.scales[rows])
        low, high = _exact_scales(part, gate, up, n)
        e = _bits(float8_swiglu(part, gate, up).scales).double() - 127.0
        assert bool(((e == low) | (e == high)).all())
