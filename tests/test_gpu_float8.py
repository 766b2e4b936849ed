"""8-bit floating point on the GPU: each operator against its definition in 64 bits, over types, sizes, strides and numbers
that are not finite."""

from __future__ import annotations

import pytest
import torch

from llmopt.quantization import (Float8Tensor, float8_linear, float8_swiglu, quantize_float8, rmsnorm_float8)
from oracle import float8_oracle as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _x(gen, rows, k, dtype=torch.float32):
    gain = torch.where(torch.rand(k, generator=gen, device="cuda") > 0.95, 8.0, 1.0)
    return (torch.randn(rows, k, generator=gen, device="cuda") * gain).to(dtype)


def _activations(gen, rows, k):
    return quantize_float8(_x(gen, rows, k))


def _weight(gen, n, k):
    return quantize_float8(torch.randn(n, k, generator=gen, device="cuda") * 0.02, block_rows=128)


def _bits(t):
    return t.view(torch.int8)


# ---- quantizing ------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 7), (1, 128), (3, 129), (1, 4096), (130, 1000), (129, 2056), (17, 5001), (257, 2816)])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantizing_is_the_hosts_bit_for_bit(dtype, rows, k, block_rows):
    x = _x(_gen(1), rows, k, dtype)
    got = quantize_float8(x, block_rows)
    want = quantize_float8(x.cpu(), block_rows)
    assert torch.equal(_bits(got.scales).cpu(), _bits(want.scales))
    assert torch.equal(_bits(got.codes).cpu(), _bits(want.codes))
    oracle.check_quantized(got.codes, got.scales, x.double(), 0.0, block_rows)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantizing_strided_and_unaligned_rows(block_rows):
    big = _x(_gen(2), 140, 1100, torch.bfloat16)
    for x in (big[:, 3:1003], big[::2, :1024], big[:, :1000], big.t()[:300], big[5:6, 8:520]):
        got, want = quantize_float8(x, block_rows), quantize_float8(x.cpu(), block_rows)
        assert torch.equal(_bits(got.scales).cpu(), _bits(want.scales)) and torch.equal(_bits(got.codes).cpu(), _bits(want.codes))
    x = big.view(7, 20, 1100)
    if block_rows == 1:
        got = quantize_float8(x)
        assert got.codes.shape == x.shape and got.scales.shape == (7, 20, 9)
        assert torch.equal(_bits(got.codes).view(140, 1100), _bits(quantize_float8(big).codes))


@pytest.mark.parametrize("block_rows", [1, 128])
def test_zeros_the_smallest_the_largest_and_what_is_not_finite(block_rows):
    x = torch.zeros(6, 640, device="cuda")
    x[0, :128] = 2.0**-140
    x[1, 130] = 3e38
    x[2, 300] = float("inf")
    x[3, 400] = float("-inf")
    x[4, 600] = float("nan")
    x[5, 5], x[5, 6] = 2.0**-118, -(2.0**-126)
    got, want = quantize_float8(x, block_rows), quantize_float8(x.cpu(), block_rows)
    assert torch.equal(_bits(got.scales).cpu(), _bits(want.scales)) and torch.equal(_bits(got.codes).cpu(), _bits(want.codes))
    assert int((got.scales.view(torch.uint8) == 255).sum()) == 3
    if block_rows == 1:
        assert torch.equal(got.dequantize()[5, :8], x[5, :8])
        assert not bool(got.dequantize()[0].any())  # 2^-140 is 2^-13 of the smallest scale, the smallest code 2^-9
        assert bool(got.dequantize()[2, 256:384].isnan().all()) and not bool(got.dequantize()[2, :256].isnan().any())


def test_magnitudes_next_to_a_scales_border():
    """448 2^e and one step of fp32 either side of it, over all exponents."""
    top = torch.ldexp(torch.tensor(448.0), torch.arange(-134, 119))
    x = torch.stack([top, torch.nextafter(top, top * 2), torch.nextafter(top, top / 2)], 1).reshape(-1, 1).cuda()
    got = quantize_float8(x)
    assert torch.equal(got.scales.double(), oracle.scales_of(x.double(), 1))
    assert torch.equal(got.dequantize()[::3], x[::3])


def test_values_next_to_a_codes_border():
    """Halfway between two codes and one step of fp32 either side of it."""
    codes = torch.arange(0, 127, dtype=torch.uint8).view(F8).float()
    mid = (codes[:-1] + codes[1:]) / 2
    x = torch.stack([mid, torch.nextafter(mid, mid + 1), torch.nextafter(mid, mid - 1)])
    x = torch.nn.functional.pad(x, (0, 2), value=448.0)  # the scale is 1
    x = torch.cat([x, -x]).cuda()
    got = quantize_float8(x)
    assert bool((got.scales.float() == 1).all())
    assert torch.equal(_bits(got.codes).cpu(), _bits(x.cpu().to(F8)))


# ---- RMSNorm ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (1, 8), (5, 127), (1, 1024), (3, 1000), (2, 4096), (33, 2816), (2, 8192), (2, 16400), (1, 40000)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(dtype, rows, hidden, residual):
    gen = _gen(3)
    x, r = _x(gen, rows, hidden, dtype), _x(gen, rows, hidden, dtype)
    weight = (1 + 0.1 * torch.randn(hidden, generator=gen, device="cuda")).to(dtype)
    out, h = rmsnorm_float8(x, weight, 1e-5, residual=r if residual else None)
    stream = r + x if residual else x
    assert torch.equal(h, stream)
    h64 = stream.double()
    y = h64 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + 1e-5) * weight.double()
    # fp32: a sum of positive terms is off by a step of 2^-24 for each addition on an element's way (a thread's own, at
    # most hidden / 256, and 10 across threads), half of it after the root, and 8 more operations
    oracle.check_quantized(out.codes, out.scales, y, y.abs() * ((hidden / 512 + 13) * 2.0**-24))


def test_norm_in_place_and_of_strided_rows():
    gen = _gen(4)
    big, r = _x(gen, 40, 1200, torch.bfloat16), _x(gen, 40, 1024, torch.bfloat16)
    weight = torch.ones(1024, dtype=torch.bfloat16, device="cuda")
    for x in (big[:, :1024], big[:, 5:1029]):
        out, h = rmsnorm_float8(x, weight, 1e-5, residual=r)
        want, h2 = rmsnorm_float8(x.contiguous(), weight, 1e-5, residual=r)
        assert torch.equal(h, h2)
        assert torch.equal(_bits(out.scales), _bits(want.scales)) and torch.equal(_bits(out.codes), _bits(want.codes))
    out, h = rmsnorm_float8(big[:, :1024].view(4, 10, 1024), weight, 1e-5, residual=r.view(4, 10, 1024))
    assert h.shape == out.codes.shape == (4, 10, 1024) and out.scales.shape == (4, 10, 8)


@pytest.mark.parametrize("hidden", [1024, 1000])
def test_norm_of_a_row_that_is_not_finite(hidden):
    x = torch.ones(4, hidden, dtype=torch.bfloat16, device="cuda")
    x[1, 3], x[2, 500] = float("inf"), float("nan")
    weight = torch.ones(hidden, dtype=torch.bfloat16, device="cuda")
    out, _ = rmsnorm_float8(x, weight, 1e-5)
    host, _ = rmsnorm_float8(x.cpu(), weight.cpu(), 1e-5)
    bad = out.dequantize().isnan()
    assert torch.equal(bad.cpu(), host.dequantize().isnan())
    assert not bool(bad[0].any() or bad[3].any()) and bool(bad[2].all())


# ---- products --------------------------------------------------------------------------------------

SHAPES = [  # tokens, N, K
    (1, 1, 1), (1, 16, 128), (1, 6144, 4096), (2, 100, 48), (3, 1536, 1040), (5, 4096, 14336), (8, 130, 272), (16, 1024, 4096),
    (17, 5632, 1024), (31, 257, 4112), (32, 4096, 4096), (33, 2816, 1024), (48, 640, 2816), (64, 28672, 256), (65, 1000, 400),
    (96, 512, 4096), (127, 1536, 1040), (128, 1024, 1024), (129, 4096, 144), (200, 3584, 4096), (255, 384, 14336),
    (256, 256, 512), (257, 2048, 640), (511, 300, 2064), (777, 1536, 1040), (1025, 640, 1024), (2000, 1160, 256),
]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype,bias", [(torch.bfloat16, False), (torch.float16, True)])
def test_linear(m, n, k, dtype, bias):
    gen = _gen(5)
    x, w = _activations(gen, m, k), _weight(gen, n, k)
    b = torch.randn(n, generator=gen, device="cuda").to(dtype) if bias else None
    y = float8_linear(x, w, b, dtype)
    assert y.shape == (m, n) and y.dtype == dtype
    _check_product(y, x, w, b)


def _check_product(y, x, w, bias=None):
    want, off = oracle.product(oracle.numbers(x.codes, x.scales, 1), oracle.numbers(w.codes, w.scales, 128))
    if bias is not None:
        want = want + bias.double()
        off = off + want.abs() * 2.0**-24
    half = torch.finfo(y.dtype).eps / 2
    least = torch.finfo(y.dtype).tiny * half  # half a step of the smallest numbers
    err = (y.double() - want).abs()
    assert bool((err <= off + (want.abs() + off) * half + least).all())
    # and their typical size, which a lost column or scale would show in: 2.6e-5 from the matrix cores' dropped bits (a
    # third of that again for other inputs), and roundings to 16 bits, evenly spread over a step of at most 2 half / sqrt(12)
    assert float(err.norm()) <= float(want.norm()) * (4e-5 + half * 1.2) + least * err.numel() ** 0.5


@pytest.mark.parametrize("k", [1, 5, 100, 1001])
@pytest.mark.parametrize("m", [1, 70])
def test_linear_of_rows_that_are_no_multiple_of_16_bytes(m, k):
    gen = _gen(6)
    x, w = _activations(gen, m, k), _weight(gen, 200, k)
    _check_product(float8_linear(x, w, dtype=torch.float16), x, w)


@pytest.mark.parametrize("m", [1, 9, 40, 100, 300, 1100])
def test_linear_of_strided_and_unaligned_operands(m):
    """The same numbers in any layout give the same bits where the rows stay aligned, and a result as near where not."""
    gen = _gen(7)
    x, w = _activations(gen, m, 1024), _weight(gen, 384, 1024)
    y = float8_linear(x, w)
    wide = torch.zeros(m, 1104, dtype=torch.int8, device="cuda")
    for at in (0, 16, 5):
        wide[:, at : at + 1024] = _bits(x.codes)
        codes = wide.view(F8)[:, at : at + 1024]
        scales = torch.nn.functional.pad(_bits(x.scales), (1, 2)).view(E8)[:, 1:9]
        z = float8_linear(Float8Tensor(codes, scales), w)
        if at % 16 == 0:
            assert torch.equal(z, y)
        else:
            _check_product(z, x, w)
    z = float8_linear(Float8Tensor(x.codes.view(m, 1, 1024), x.scales.view(m, 1, 8)), w)
    assert torch.equal(z.view(m, 384), y)


@pytest.mark.parametrize("m", [1, 20, 100, 600])
def test_what_is_not_finite_stays_in_its_rows(m):
    gen = _gen(8)
    x, w = _activations(gen, m, 1024), _weight(gen, 300, 1024)
    clean = float8_linear(x, w)
    x.scales.view(torch.uint8)[m // 2, 3] = 255
    y = float8_linear(x, w)
    rows = torch.arange(m, device="cuda") != m // 2
    assert bool(y[m // 2].isnan().all()) and torch.equal(y[rows], clean[rows])
    x.scales.view(torch.uint8)[m // 2, 3] = 120
    clean = float8_linear(x, w)
    w.scales.view(torch.uint8)[1, 2] = 255
    y = float8_linear(x, w)
    assert bool(y[:, 128:256].isnan().all())
    assert torch.equal(y[:, :128], clean[:, :128]) and torch.equal(y[:, 256:], clean[:, 256:])
    _bits(w.codes)[290, 7] = 0x7F  # a NaN code
    assert bool(float8_linear(x, w)[:, 290].isnan().all())


def test_scales_from_the_smallest_to_the_largest():
    """Exponents far apart in one row: the products of far scales meet in range."""
    gen = _gen(11)
    for m in (1, 40, 300):
        x, w = _activations(gen, m, 512), _weight(gen, 256, 512)
        x.scales.view(torch.uint8)[:] = torch.tensor([0, 60, 127, 240], dtype=torch.uint8, device="cuda")
        w.scales.view(torch.uint8)[:] = torch.tensor([250, 190, 120, 8], dtype=torch.uint8, device="cuda")
        _check_product(float8_linear(x, w), x, w)


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 14336, 4096), (4, 300, 1040), (7, 2816, 1024), (16, 128, 512), (33, 1000, 784),
                                   (64, 640, 4096), (65, 256, 128), (130, 129, 1024), (200, 2816, 1024), (300, 1280, 2048),
                                   (1030, 700, 272), (3, 50, 77)])
def test_swiglu(m, n, k):
    gen = _gen(9)
    x, gate, up = _activations(gen, m, k), _weight(gen, n, k), _weight(gen, n, k)
    gate.scales.view(torch.uint8).add_(2)  # gates of some units
    out = float8_swiglu(x, gate, up)
    want, off = oracle.swiglu(oracle.numbers(x.codes, x.scales, 1), oracle.numbers(gate.codes, gate.scales, 128),
                              oracle.numbers(up.codes, up.scales, 128))
    assert out.codes.shape == (m, n)
    oracle.check_quantized(out.codes, out.scales, want, off)


def test_no_tokens_no_features_no_columns():
    w = _weight(_gen(10), 40, 256)
    x = quantize_float8(torch.zeros(0, 256, device="cuda"))
    assert float8_linear(x, w).shape == (0, 40) and float8_swiglu(x, w, w).codes.shape == (0, 40)
    out, h = rmsnorm_float8(torch.zeros(0, 256, dtype=torch.bfloat16, device="cuda"),
                            torch.ones(256, dtype=torch.bfloat16, device="cuda"), 1e-5)
    assert out.codes.shape == (0, 256) and h.shape == (0, 256)
    empty = quantize_float8(torch.zeros(3, 0, device="cuda"))
    none = quantize_float8(torch.zeros(5, 0, device="cuda"), block_rows=128)
    bias = torch.arange(5, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(float8_linear(empty, none, bias), bias.expand(3, 5))
