"""8-bit floating point at the edges of what its entry points take."""

from __future__ import annotations

import pytest
import torch

from llmopt.kernels import _lib
from llmopt.quantization import Float8Tensor, float8_linear, float8_swiglu, quantize_float8, rmsnorm_float8
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


def _at_a_border(gen, gate, up, k):
    """Of many tokens, one whose largest magnitude of the block's 128 features lies within 1e-4 of a border, but not within 2e-5, and
    one that is far from it. Of the larger half of all: their sums do not cancel."""
    x = quantize_float8(torch.randn(65536, k, generator=gen, device="cuda"))
    amax = oracle.swiglu(_numbers(x), _numbers(gate), _numbers(up))[0].abs().amax(1)
    off = torch.log2(amax / 448.0)
    off = torch.where(amax > amax.median(), (off - off.round()).abs(), 0.0)
    near = torch.where(off > 3e-5, off, 1.0).argmin()
    assert float(off[near]) < 1.4e-4
    return [Float8Tensor(x.codes[t : t + 1], x.scales[t : t + 1]) for t in (near, off.argmax())]


def _repeated(t, rows):
    """The rows of activations, or the block of 128 rows of a weight, over and over."""
    times = rows // t.codes.shape[0]
    codes, scales = (part.view(torch.uint8).repeat(times, 1).view(part.dtype) for part in (t.codes, t.scales))
    return Float8Tensor(codes, scales, t.block_rows)


def _us(call, calls=5):
    best = float("inf")
    for _ in range(4):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(calls):
            call()
        end.record()
        end.synchronize()
        best = min(best, start.elapsed_time(end) * 1e3 / calls)
    return best


@pytest.mark.parametrize("tokens", [16, 200, 1024, 4096])
def test_equal_tokens_next_to_a_border(tokens):
    """A batch of one token, and a weight of one block, over and over: all groups are next to the border together. They have the scale
    of the exact sums, all the same codes, and take about as long as other tokens."""
    gen, k, n = _gen(32), 1024, 128 * 64
    gate, up = _weight(gen, 128, k), _weight(gen, 128, k)
    near, far = _at_a_border(gen, gate, up, k)
    low, high = _exact_scales(near, gate, up, 128)
    assert torch.equal(low, high)
    near, far, gate, up = _repeated(near, tokens), _repeated(far, tokens), _repeated(gate, n), _repeated(up, n)
    out = float8_swiglu(near, gate, up)
    assert bool((_bits(out.scales).double() - 127.0 == low).all())
    assert torch.equal(_bits(out.codes), _bits(out.codes)[:1].expand(tokens, n))
    us = [_us(lambda x=x: float8_swiglu(x, gate, up)) for x in (near, far)]
    assert us[0] < 2 * us[1] + 10, us


@pytest.mark.parametrize("tokens", [1, 40, 256, 2048])
def test_equal_features_next_to_a_border(tokens):
    """Every feature of a weight the same: all of a group's numbers are next to the border. Not all of them are summed again, and the
    time stays bounded: a wave takes at most 16 sums for a tile."""
    gen, k, n = _gen(33), 1024, 1024
    gate, up = (_repeated(quantize_float8(torch.randn(1, k, generator=gen, device="cuda") * 0.05), n) for _ in range(2))
    gate, up = (quantize_float8(t.dequantize(), block_rows=128) for t in (gate, up))
    near, far = _at_a_border(gen, Float8Tensor(gate.codes[:128], gate.scales[:1], 128), Float8Tensor(up.codes[:128], up.scales[:1], 128), k)
    near, far = _repeated(near, tokens), _repeated(far, tokens)
    out = float8_swiglu(near, gate, up)
    oracle.check_quantized(out.codes, out.scales, *oracle.swiglu(_numbers(near), _numbers(gate), _numbers(up)))
    us = [_us(lambda x=x: float8_swiglu(x, gate, up)) for x in (near, far)]
    assert us[0] < 10 * us[1] + 50, us


# ---- no columns, tokens or features ------------------------------------------------------------------


@pytest.mark.parametrize("lead", [(), (3,), (0,), (2, 3), (2, 0)])
def test_no_columns_no_tokens_no_features(lead):
    x, w = quantize_float8(torch.zeros(*lead, 0, device="cuda")), quantize_float8(torch.zeros(5, 0, device="cuda"), block_rows=128)
    assert x.codes.shape == x.scales.shape == (*lead, 0) and w.scales.shape == (1, 0)
    bias = torch.arange(5, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(float8_linear(x, w, bias), bias.expand(*lead, 5))
    act = float8_swiglu(x, w, w)
    assert act.codes.shape == (*lead, 5) and act.scales.shape == (*lead, 1) and not bool(act.dequantize().any())
    zeros = torch.zeros(*lead, 0, dtype=torch.bfloat16, device="cuda")
    out, h = rmsnorm_float8(zeros, zeros.new_zeros(0), 1e-5, residual=zeros)
    assert out.codes.shape == h.shape == (*lead, 0)
    x, none = quantize_float8(torch.ones(*lead, 200, device="cuda")), quantize_float8(torch.zeros(0, 200, device="cuda"), block_rows=128)
    assert float8_linear(x, none).shape == (*lead, 0) and float8_swiglu(x, none, none).scales.shape == (*lead, 0)


# ---- outputs in place ---------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,hidden,ld", [(1, 8, 8), (5, 1024, 1024), (3, 1000, 1003), (40, 4096, 4100), (2, 8192, 8200), (3, 16400, 16400)])
@pytest.mark.parametrize("place", ["x", "residual"])
def test_the_norms_stream_in_place(dtype, rows, hidden, ld, place):
    """``h_out`` may be ``x`` or the residual: what comes of it is what comes of a stream of its own, and what lies between the rows is
    left as it was."""
    gen, lib, across = _gen(41), _lib.load_library(), -(-hidden // 128)
    wide = [torch.randn(rows, ld, generator=gen, device="cuda").to(dtype) for _ in range(2)]
    x, residual = (t[:, :hidden] for t in wide)
    weight = (1 + 0.1 * torch.randn(hidden, generator=gen, device="cuda")).to(dtype)
    want, stream = rmsnorm_float8(x, weight, 1e-5, residual=residual)
    before = [t.clone() for t in wide]
    h = wide[0] if place == "x" else wide[1]
    codes = torch.empty(rows, hidden, dtype=F8, device="cuda")
    scales = torch.empty(rows, across, dtype=E8, device="cuda")
    _lib.call(lib.llmopt_f8_rmsnorm(x.data_ptr(), ld, residual.data_ptr(), ld, h.data_ptr(), ld, weight.data_ptr(), codes.data_ptr(),
                                    hidden, scales.data_ptr(), across, rows, hidden, 1e-5, _lib.DTYPE_CODES[dtype], _stream()),
              "llmopt_f8_rmsnorm")
    assert torch.equal(_bits(codes), _bits(want.codes)) and torch.equal(_bits(scales), _bits(want.scales))
    assert torch.equal(h[:, :hidden], stream)
    assert all(torch.equal(t[:, hidden:], b[:, hidden:]) for t, b in zip(wide, before))
    other = 1 if place == "x" else 0
    assert torch.equal(wide[other], before[other])


# ---- each kernel's typical error ------------------------------------------------------------------------


def _near_product(x, w):
    """``x w^T`` in 64 bits, and how far sums of products of either sign are off. Each of the seven smaller products of eight neighbouring ones
    loses less than 2^-13 of the largest, in either direction: by Hoeffding's bound a sum is off by more than t 2^-13 root(7 times the
    sum of the squares of the largest ones) in 2 exp(-t^2 / 2) of all cases, 5e-11 at t = 7; and the squares of all products are
    no fewer. So 7 root 7 2^-13 = 2.3e-3 of the root of the sum of squares, a tenth more for the fp32 additions."""
    return x @ w.t().contiguous(), 2.5e-3 * torch.sqrt((x * x) @ (w * w).t().contiguous())


def _check_near(y, want, off):
    half = torch.finfo(y.dtype).eps / 2
    assert bool(((y.double() - want).abs() <= off + (want.abs() + off) * half + 2.0**-25).all())  # half of fp16's least step


LINEAR = [
    # the few-token kernel
    (1, 6144, 4096), (4, 4096, 14336), (16, 1024, 4096), (17, 40, 16), (31, 300, 2064), (32, 1000, 4096), (33, 130, 4112), (150, 100, 2048),
    # the tiles, whole and in parts of K
    (1036, 16, 16), (8249, 16, 1968), (1036, 16, 1664), (1045, 16, 3680), (32, 4096, 14336), (130, 22445, 16), (8886, 261, 13728),
    (8809, 16, 7456), (7202, 16, 5056), (130, 20409, 16), (130, 10691, 10160), (17, 15263, 2320), (133, 28530, 400), (66, 27201, 7936),
    (65, 6387, 13952), (258, 22201, 16), (526, 21875, 272), (513, 14350, 6528), (261, 25258, 912), (534, 26166, 272),
    # rows of any alignment
    (70, 200, 1001), (1, 200, 77)]


@pytest.mark.parametrize("m,n,k", LINEAR)
def test_a_products_error_is_that_of_its_dropped_bits(m, n, k):
    """Sixteen columns less would show, in any kernel: of 14336 they are 3 % of a typical sum."""
    gen = _gen(42)
    x, w = quantize_float8(torch.randn(m, k, generator=gen, device="cuda")), _weight(gen, n, k)
    _check_near(float8_linear(x, w, dtype=torch.float16), *_near_product(_numbers(x), _numbers(w)))


@pytest.mark.parametrize("m,n,k", [(1, 6144, 4096), (16, 4096, 14336), (32, 1536, 1024), (200, 3584, 4096), (777, 1536, 1040), (2000, 4096, 4096)])
@pytest.mark.parametrize("share,gain", [(0.01, 8.0), (0.002, 100.0), (0.001, 1000.0)])
def test_a_product_where_a_few_channels_are_strong(m, n, k, share, gain):
    """A strong channel's product takes bits of the seven beside it: up to 1e-4 of a typical sum where it is all of it, half of what
    a rounding to fp16 brings. The largest products of eight are as independent as their signs, and a product's dropped bits spread
    evenly up to 2^-13 of the largest: root(7 / 3) 2^-13 = 1.9e-4 of their root of squares, which the sums have for their own."""
    gen = _gen(43)
    x, w = quantize_float8(_strong(gen, m, k, share, gain)), quantize_float8(torch.randn(n, k, generator=gen, device="cuda") * 0.004, block_rows=128)
    want, off = _near_product(_numbers(x), _numbers(w))
    y = float8_linear(x, w, dtype=torch.float16)
    _check_near(y, want, off)
    err = (y.double() - want).norm()
    assert float(err) <= float(want.norm()) * (2e-4 + 2.0**-11) + 2.0**-25 * want.numel() ** 0.5


GATED = [
    # the few-token kernel, the tiles, several one after the other, rows of any alignment
    (1, 14336, 4096), (7, 2816, 1024), (32, 1000, 4096), (50, 260, 4112), (300, 1280, 2048), (200, 14336, 4096), (700, 130, 272),
    (1035, 17, 400), (8262, 129, 272), (130, 16428, 400), (262, 12981, 928), (260, 16758, 400), (264, 22740, 272), (2048, 2816, 1024),
    (70, 200, 1001)]


@pytest.mark.parametrize("m,n,k", GATED)
def test_the_gated_codes_are_the_nearest_but_for_dropped_bits(m, n, k):
    """Sums are off by some 1e-4 of a number at most and a code's step is a twelfth of it, so one code in some hundreds is not the nearest to
    the exact number: in no 16 tokens by 64 features more than 3 %. Without 16 columns of the product a third would be."""
    gen = _gen(44)
    x, gate, up = quantize_float8(torch.randn(m, k, generator=gen, device="cuda")), _weight(gen, n, k), _weight(gen, n, k)
    out = float8_swiglu(x, gate, up)
    (g, dg), (u, du) = (_near_product(_numbers(x), _numbers(w)) for w in (gate, up))
    s = g * torch.sigmoid(g)
    want = s * u
    oracle.check_quantized(out.codes, out.scales, want, 1.1 * dg * (u.abs() + du) + s.abs() * du + want.abs() * (16 + 4 * g.abs()) * 2.0**-24)
    v = want / oracle.spread(out.scales.double(), 1, want.shape)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0**-6))) - 3)  # three fraction bits
    other = (torch.round(v / step) * step).clamp(-448, 448) != out.codes.double()
    other = torch.nn.functional.pad(other.double(), (0, -n % 64, 0, -m % 16))
    share = other.view(-(-m // 16), 16, -(-n // 64), 64).sum((1, 3)) / (min(m, 16) * min(n, 64))
    assert float(share.max()) <= 0.03 + 1 / (min(m, 16) * min(n, 64)) * 3, float(share.max())


# ---- layouts, and what is not finite --------------------------------------------------------------------


@pytest.mark.parametrize("m", [3, 40, 300])
def test_operands_of_any_layout(m):
    """Columns of a transposed tensor, one prompt expanded to two, tokens in front of prompts, a bias that is every other number."""
    gen = _gen(51)
    x, w = quantize_float8(torch.randn(m, 256, generator=gen, device="cuda")), _weight(gen, 384, 256)
    y, act = float8_linear(x, w), float8_swiglu(x, w, w)
    xt = Float8Tensor(x.codes.t().contiguous().t(), x.scales.t().contiguous().t())
    wt = Float8Tensor(w.codes.t().contiguous().t(), w.scales.t().contiguous().t(), 128)
    assert torch.equal(float8_linear(xt, wt), y)
    assert torch.equal(_bits(float8_swiglu(xt, wt, w).codes), _bits(act.codes))
    two = Float8Tensor(x.codes.expand(2, m, 256), x.scales.expand(2, m, 2))
    want = float8_linear(Float8Tensor(two.codes.contiguous(), two.scales.contiguous()), w)
    assert torch.equal(float8_linear(two, w), want)
    swapped = Float8Tensor(two.codes.transpose(0, 1), two.scales.transpose(0, 1))
    assert torch.equal(float8_linear(swapped, w), want.transpose(0, 1))
    bias = torch.randn(768, generator=gen, device="cuda").bfloat16()[::2]
    assert torch.equal(float8_linear(x, w, bias), float8_linear(x, w, bias.contiguous()))


@pytest.mark.parametrize("m,n,k", [(3, 300, 256), (40, 300, 1024), (300, 4000, 1024), (5, 50, 77), (700, 2816, 1024)])
def test_what_is_not_finite_stays_in_its_groups_of_the_gated_product(m, n, k):
    """A token's NaN scale, a feature's NaN code and a block's NaN scale: the groups that read as NaN are the host's, their codes 0."""
    gen = _gen(52)
    x, gate, up = quantize_float8(torch.randn(m, k, generator=gen, device="cuda")), _weight(gen, n, k), _weight(gen, n, k)
    clean = float8_swiglu(x, gate, up)
    _bits(x.scales)[m // 2, 0] = 255
    _bits(up.codes)[17, 3] = 0x7F
    if n > 256:
        _bits(gate.scales)[1, 0] = 255
    out = float8_swiglu(x, gate, up)
    host = float8_swiglu(x.to("cpu"), gate.to("cpu"), up.to("cpu"))
    bad = out.dequantize().isnan()
    assert torch.equal(bad.cpu(), host.dequantize().isnan()) and not bool(_bits(out.codes)[bad].any())
    assert torch.equal(_bits(out.codes)[~bad], _bits(clean.codes)[~bad])
    large = quantize_float8(torch.full((m, 128), 1e20, device="cuda"))
    w = quantize_float8(torch.full((200, 128), 1e20, device="cuda"), block_rows=128)
    assert bool(float8_linear(large, w).isinf().all()) and bool(float8_swiglu(large, w, w).dequantize().isnan().all())
