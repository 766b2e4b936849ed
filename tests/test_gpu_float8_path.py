"""The steps in 8-bit floating point as a decoder runs them, on the GPU: one after the other with each checked on what it was
given, captured and replayed, on other streams, through the general host path, at sizes whose offsets pass 32 bits, and in the
model and generator."""

from __future__ import annotations

import pytest
import torch

from llmopt.kernels import _lib, float8_ops
from llmopt.model import DecoderOnlyModel, GreedyGenerator, ModelConfig, fuse_projections_
from llmopt.quantization import (Float8Linear, Float8SwiGLU, Float8Tensor, FusedFloat8Linear, float8_linear, float8_swiglu,
                                 quantize_float8, quantize_model_float8_, rmsnorm_float8)
from oracle import float8_oracle as oracle

pytestmark = pytest.mark.gpu

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _bits(t):
    return t.view(torch.uint8)


def _weight(gen, n, k):
    return quantize_float8(torch.randn(n, k, generator=gen, device="cuda") * 0.05, block_rows=128)


def _numbers(t):
    return oracle.numbers(t.codes, t.scales, t.block_rows)


def _equal(a, b):
    return torch.equal(_bits(a.codes), _bits(b.codes)) and torch.equal(_bits(a.scales), _bits(b.scales))


def _check_16(y, want, off):
    half = torch.finfo(y.dtype).eps / 2
    assert bool(((y.double() - want).abs() <= off + (want.abs() + off) * half + 2.0**-30).all())


# ---- a layer's steps --------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens", [1, 5, 16, 17, 64, 200, 513])
@pytest.mark.parametrize("hidden,wide", [(1024, 2816), (528, 400)])
def test_a_layers_steps_one_after_the_other(tokens, hidden, wide):
    """Norm with the residual, gate and up, down: each on what the one in front of it gave."""
    gen = _gen(1)
    x, residual = _randn(gen, tokens, hidden), _randn(gen, tokens, hidden)
    norm = (1 + 0.1 * torch.randn(hidden, generator=gen, device="cuda")).bfloat16()
    gate, up, down = _weight(gen, wide, hidden), _weight(gen, wide, hidden), _weight(gen, hidden, wide)
    normed, stream = rmsnorm_float8(x, norm, 1e-6, residual=residual)
    assert torch.equal(stream, residual + x)
    h = stream.double()
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * norm.double()
    oracle.check_quantized(normed.codes, normed.scales, y, y.abs() * ((hidden / 512 + 13) * 2.0**-24))
    act = float8_swiglu(normed, gate, up)
    oracle.check_quantized(act.codes, act.scales, *oracle.swiglu(_numbers(normed), _numbers(gate), _numbers(up)))
    out = float8_linear(act, down)
    _check_16(out, *oracle.product(_numbers(act), _numbers(down)))


@pytest.mark.parametrize("tokens", [3, 40, 300])
def test_layers_are_their_operators(tokens):
    gen = _gen(2)
    weights = [_weight(gen, n, 512) for n in (256, 128, 128)]
    x = _randn(gen, tokens, 512)
    q = quantize_float8(x)
    parts = [Float8Linear(w) for w in weights]
    fused = FusedFloat8Linear(parts)
    for y, p, w in zip(fused(x), parts, weights):
        want, off = oracle.product(_numbers(q), _numbers(w))
        _check_16(y, want, off)
        _check_16(p(q), want, off)
        assert torch.equal(p(x), p(q))
    gate, up = Float8Linear(_weight(gen, 300, 512)), Float8Linear(_weight(gen, 300, 512))
    assert _equal(Float8SwiGLU(gate, up)(x), float8_swiglu(q, gate.weight_tensor(), up.weight_tensor()))


@pytest.mark.parametrize("tokens", [2, 100])
def test_a_gradient_on_the_device(tokens):
    gen = _gen(3)
    layer = Float8Linear(_weight(gen, 200, 300), torch.zeros(200, device="cuda"))
    x, seed = _randn(gen, tokens, 300).requires_grad_(), _randn(gen, tokens, 200)
    layer(x).backward(seed)
    w = _numbers(layer.weight_tensor())
    want, terms = seed.double() @ w, seed.double().abs() @ w.abs()
    # fp32 sums of 200 terms, rounded to bf16
    assert bool(((x.grad.double() - want).abs() <= terms * 200 * 2.0**-23 + want.abs() * 2.0**-8 * 1.01).all())
    h = rmsnorm_float8(x, torch.ones(300, dtype=torch.bfloat16, device="cuda"), 1e-6, residual=seed.new_ones(tokens, 300))[1]
    assert h.requires_grad
    with torch.no_grad():
        assert not layer(x).requires_grad


# ---- captured, on other streams, in the general host path ----------------------------------------------


@pytest.mark.parametrize("tokens", [1, 33, 300])
def test_two_captured_graphs_replayed_with_new_inputs(tokens):
    """Both hold a workspace of one pool; eager calls and each other's replays come in between."""
    gen = _gen(4)
    gate, up, down = _weight(gen, 384, 512), _weight(gen, 384, 512), _weight(gen, 512, 384)
    norm = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    x, residual = _randn(gen, tokens, 512), _randn(gen, tokens, 512)

    def step(a, b):
        normed, stream = rmsnorm_float8(a, norm, 1e-6, residual=b)
        return float8_linear(float8_swiglu(normed, gate, up), down), stream, quantize_float8(stream).scales

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        step(x, residual)
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side, pool=graphs[0][0].pool() if graphs else None):
                graphs.append((graph, step(x, residual)))
    torch.cuda.current_stream().wait_stream(side)
    for turn in range(3):
        x.copy_(_randn(gen, tokens, 512))
        residual.copy_(_randn(gen, tokens, 512))
        want = step(x, residual)
        for graph, got in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(_bits(got[2]), _bits(want[2]))


def test_two_streams_at_once():
    gen = _gen(5)
    w = _weight(gen, 512, 2048)
    xs = [quantize_float8(_randn(gen, 40, 2048)) for _ in range(2)]
    want = [float8_linear(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(float8_linear(xs[i], w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


@pytest.mark.parametrize("tokens", [1, 20, 200])
def test_the_general_host_path_gives_the_same_bits(tokens, monkeypatch):
    gen = _gen(6)
    x, residual = _randn(gen, 2, tokens, 528), _randn(gen, 2, tokens, 528)
    norm = torch.ones(528, dtype=torch.bfloat16, device="cuda")
    gate, up = _weight(gen, 300, 528), _weight(gen, 300, 528)
    bias = _randn(gen, 300)

    def all_of_it():
        n, h = rmsnorm_float8(x, norm, 1e-6, residual=residual)
        plain, same = rmsnorm_float8(x, norm, 1e-6)
        assert same is x
        q = quantize_float8(x)
        made = Float8Tensor(q.codes, q.scales)
        block = quantize_float8(x[0], block_rows=128)
        act = float8_swiglu(n, gate, up)
        return [n.codes, n.scales, h, plain.codes, plain.scales, q.codes, q.scales, block.codes, block.scales, act.codes,
                act.scales, float8_linear(made, gate, bias), float8_linear(n, up, dtype=torch.float16)]

    native = all_of_it()
    assert float8_ops.native() is _lib.load_binding()
    monkeypatch.setattr(float8_ops, "load_binding", lambda: None)
    for a, b in zip(native, all_of_it()):
        assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a.view(torch.int16 if a.element_size() == 2 else torch.uint8), b.view(torch.int16 if b.element_size() == 2 else torch.uint8))


def test_refusals_on_the_device():
    gen = _gen(7)
    x, w = quantize_float8(_randn(gen, 4, 256)), _weight(gen, 40, 256)
    with pytest.raises(RuntimeError, match="same device"):
        float8_linear(x, w.to("cpu"))
    with pytest.raises(RuntimeError, match="same device"):
        Float8Tensor(x.codes, x.scales.cpu())
    with pytest.raises(RuntimeError, match="cannot be multiplied"):
        float8_linear(x, _weight(gen, 40, 272))
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        float8_linear(x, w, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="same dtype"):
        float8_linear(x, w, torch.zeros(40, dtype=torch.float16, device="cuda"))
    with pytest.raises(ValueError, match="scales"):
        Float8Tensor(x.codes, x.scales[:, :1])
    with pytest.raises(ValueError, match="different shapes"):
        float8_swiglu(x, w, _weight(gen, 41, 256))
    with pytest.raises(ValueError, match="weight"):
        rmsnorm_float8(_randn(gen, 4, 256), torch.ones(255, dtype=torch.bfloat16, device="cuda"), 1e-6)
    with pytest.raises(TypeError, match="floating-point"):
        quantize_float8(torch.zeros(3, 4, dtype=torch.int32, device="cuda"))


def test_other_types_of_a_norm_run_in_torch():
    gen = _gen(8)
    x, weight = torch.randn(3, 300, generator=gen, device="cuda", dtype=torch.float64), torch.ones(300, device="cuda", dtype=torch.float64)
    out, h = rmsnorm_float8(x, weight, 1e-6)
    assert h is x
    oracle.check_quantized(out.codes, out.scales, x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6), x.abs() * 2.0**-17)


@pytest.mark.parametrize("m", [1, 40])
def test_a_bias_has_its_derivative(m):
    gen = _gen(27)
    x, w = quantize_float8(_randn(gen, m, 256)), _weight(gen, 40, 256)
    bias = _randn(gen, 40).requires_grad_()
    y = float8_linear(x, w, bias)
    y.sum().backward()
    assert torch.equal(bias.grad, torch.full_like(bias, m))
    with torch.no_grad():
        assert not float8_linear(x, w, bias).requires_grad
    want, off = oracle.product(_numbers(x), _numbers(w))
    _check_16(y.detach(), want + bias.detach().double(), off + (want + bias.detach().double()).abs() * 2.0**-24)


# ---- without the workspace --------------------------------------------------------------------------


def _call_linear(x, w, dtype, workspace):
    lib = _lib.load_library()
    (m, k), n = x.codes.shape, w.codes.shape[0]
    y = torch.empty(m, n, dtype=dtype, device="cuda")
    ws = torch.empty(workspace, dtype=torch.uint8, device="cuda") if workspace else None
    _lib.call(lib.llmopt_f8_linear(x.codes.data_ptr(), k, x.scales.data_ptr(), x.scales.shape[1], m, k, w.codes.data_ptr(), k,
                                   w.scales.data_ptr(), w.scales.shape[1], None, y.data_ptr(), n, n, _lib.DTYPE_CODES[dtype],
                                   None if ws is None else ws.data_ptr(), workspace, torch.cuda.current_stream().cuda_stream),
              "llmopt_f8_linear")
    return y


@pytest.mark.parametrize("m,n,k", [(17, 512, 4096), (100, 1024, 4096), (32, 300, 14336), (32, 4096, 14336), (100, 4100, 4112),
                                   (200, 3584, 4096), (6337, 134, 6944)])
def test_a_linear_with_less_workspace_than_asked_for(m, n, k):
    """The last four split K and ask for some; the narrow weights in front of them go without."""
    gen = _gen(9)
    x, w = quantize_float8(_randn(gen, m, k)), _weight(gen, n, k)
    need = _lib.load_library().llmopt_f8_linear_workspace(m, n, k)
    assert (need > 0) == (m * n > 120000)
    want, off = oracle.product(_numbers(x), _numbers(w))
    for workspace in (0, need // 2, max(0, need - 1), need):
        _check_16(_call_linear(x, w, torch.bfloat16, workspace), want, off)


@pytest.mark.parametrize("m", [1, 7, 16, 17, 80])
def test_the_gated_product_without_its_workspace(m):
    gen = _gen(10)
    x, gate, up = quantize_float8(_randn(gen, m, 1024)), _weight(gen, 300, 1024), _weight(gen, 300, 1024)
    codes, scales = torch.empty(m, 300, dtype=F8, device="cuda"), torch.empty(m, 3, dtype=E8, device="cuda")
    _lib.call(_lib.load_library().llmopt_f8_swiglu(
        x.codes.data_ptr(), 1024, x.scales.data_ptr(), 8, m, 1024, gate.codes.data_ptr(), 1024, gate.scales.data_ptr(), 8,
        up.codes.data_ptr(), 1024, up.scales.data_ptr(), 8, 300, codes.data_ptr(), 300, scales.data_ptr(), 3, None, 0,
        torch.cuda.current_stream().cuda_stream), "llmopt_f8_swiglu")
    oracle.check_quantized(codes, scales, *oracle.swiglu(_numbers(x), _numbers(gate), _numbers(up)))


# ---- every kernel that a size can lead to ------------------------------------------------------------


@pytest.mark.parametrize("m,n,k", [
    # up to 16 tokens' kernel, 32 at a time: one group of steps a wave, eight waves, and several groups
    (17, 40, 16), (31, 300, 2064), (32, 1000, 4096), (33, 130, 4112), (50, 260, 208), (150, 100, 2048), (1000, 64, 640),
    # a tile for every workgroup: 128 x 64 in 1, 2, 4 and 8 parts, then 128 x 128, 256 x 64 and 256 x 128 likewise, 256 x 256
    (1036, 16, 16), (8249, 16, 1968), (1036, 16, 1664), (1045, 16, 3680),
    (130, 22445, 16), (8886, 261, 13728), (8809, 16, 7456), (7202, 16, 5056),
    (130, 20409, 16), (130, 10691, 10160), (17, 15263, 2320), (17, 7820, 5968),
    (133, 28530, 400), (66, 27201, 7936), (6337, 134, 6944), (65, 6387, 13952),
    (258, 22201, 16),
    # several tiles one after the other
    (526, 21875, 272), (513, 14350, 6528), (261, 25258, 912), (536, 23619, 400), (534, 26166, 272)])
def test_linear_of_every_tile_and_number_of_parts(m, n, k):
    gen = _gen(21)
    x, w, bias = quantize_float8(_randn(gen, m, k)), _weight(gen, n, k), _randn(gen, n)
    want, off = oracle.product(_numbers(x), _numbers(w))
    want = want + bias.double()
    off = off + want.abs() * 2.0**-24
    y = float8_linear(x, w, bias)
    _check_16(y, want, off)
    assert torch.equal(float8_linear(x, w, bias), y)


@pytest.mark.parametrize("m,n,k", [(17, 40, 16), (31, 300, 2064), (32, 1000, 4096), (50, 260, 4112), (700, 130, 272),
                                   (1035, 17, 16), (8262, 129, 16), (130, 16428, 16),
                                   (262, 12981, 928), (260, 16758, 400), (264, 22740, 272)])
def test_the_gated_product_of_every_tile(m, n, k):
    gen = _gen(22)
    x, gate, up = quantize_float8(_randn(gen, m, k)), _weight(gen, n, k), _weight(gen, n, k)
    out = float8_swiglu(x, gate, up)
    oracle.check_quantized(out.codes, out.scales, *oracle.swiglu(_numbers(x), _numbers(gate), _numbers(up)))
    assert _equal(float8_swiglu(x, gate, up), out)


@pytest.mark.parametrize("at_once,k", [(16, 1024), (16, 2000), (512, 1024), (1024, 1024), (1024, 1000)])
def test_the_gated_products_scales_are_those_of_exact_sums(at_once, k):
    """The matrix cores' sums put one group in some 30,000 on the wrong side of a border, where its scale doubles. All are on the
    right one but where the largest magnitude is within 1e-5 of it: fp32 sums of 1000 products of random signs are off by some
    2^-24 of their typical size, 170 times less."""
    gen, m, n = _gen(26), 1024, 14336
    x, gate, up = quantize_float8(_randn(gen, m, k)), _weight(gen, n, k), _weight(gen, n, k)
    gate.scales.view(torch.uint8).add_(1)
    want, _ = oracle.swiglu(_numbers(x), _numbers(gate), _numbers(up))
    amax = want.abs().view(m, n // 128, 128).amax(2)
    low, high = (torch.ceil(torch.log2(amax * (1 + off) / 448.0)) for off in (-1e-5, 1e-5))
    for first in range(0, m, at_once):
        rows = slice(first, first + at_once)
        out = float8_swiglu(Float8Tensor(x.codes[rows], x.scales[rows]), gate, up)
        e = _bits(out.scales).double() - 127.0
        assert bool(((e == low[rows]) | (e == high[rows])).all())


@pytest.mark.parametrize("m,n,k", [(3, 40, 1040), (40, 300, 1040), (70, 4100, 4112), (300, 4100, 1040), (600, 20000, 272)])
def test_what_lies_between_and_behind_the_output_rows_is_left_as_it_was(m, n, k):
    gen = _gen(23)
    x, w = quantize_float8(_randn(gen, m, k)), _weight(gen, n, k)
    for ld in (n + 5, n + 12 + -n % 8):
        y = torch.full((m + 3, ld), 7.0, dtype=torch.bfloat16, device="cuda")
        lib = _lib.load_library()
        need = lib.llmopt_f8_linear_workspace(m, n, k)
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        _lib.call(lib.llmopt_f8_linear(x.codes.data_ptr(), k, x.scales.data_ptr(), x.scales.shape[1], m, k, w.codes.data_ptr(), k,
                                       w.scales.data_ptr(), w.scales.shape[1], None, y.data_ptr(), ld, n, 2,
                                       ws.data_ptr() if need else None, need, torch.cuda.current_stream().cuda_stream),
                  "llmopt_f8_linear")
        assert bool((y[:, n:] == 7.0).all() and (y[m:] == 7.0).all())
        assert torch.equal(y[:m, :n], float8_linear(x, w))


@pytest.mark.parametrize("m,n,k", [(3, 40, 1040), (40, 300, 1040), (70, 14336, 272), (300, 4100, 1040), (300, 20000, 272)])
def test_what_lies_between_and_behind_the_gated_rows_is_left_as_it_was(m, n, k):
    gen = _gen(24)
    x, gate, up = quantize_float8(_randn(gen, m, k)), _weight(gen, n, k), _weight(gen, n, k)
    want, across = float8_swiglu(x, gate, up), -(-n // 128)
    for ld in (n + 5, n + 16 + -n % 16):
        codes = torch.full((m + 3, ld), 77, dtype=torch.uint8, device="cuda")
        scales = torch.full((m + 3, across + 3), 78, dtype=torch.uint8, device="cuda")
        lib = _lib.load_library()
        need = lib.llmopt_f8_swiglu_workspace(m, n, k)
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        sx = x.scales.shape[1]
        _lib.call(lib.llmopt_f8_swiglu(
            x.codes.data_ptr(), k, x.scales.data_ptr(), sx, m, k, gate.codes.data_ptr(), k, gate.scales.data_ptr(), sx,
            up.codes.data_ptr(), k, up.scales.data_ptr(), sx, n, codes.data_ptr(), ld, scales.data_ptr(), across + 3,
            ws.data_ptr() if need else None, need, torch.cuda.current_stream().cuda_stream), "llmopt_f8_swiglu")
        assert bool((codes[:, n:] == 77).all() and (codes[m:] == 77).all())
        assert bool((scales[:, across:] == 78).all() and (scales[m:] == 78).all())
        assert torch.equal(codes[:m, :n], _bits(want.codes)) and torch.equal(scales[:m, :across], _bits(want.scales))


# ---- more rows than a launch counts ------------------------------------------------------------------


def test_more_rows_than_one_launch_takes():
    """Each row has a workgroup of 256, and a launch counts its work-items in 32 bits."""
    rows, cols = (1 << 24) + 5, 24
    x = torch.randn(1 << 16, cols, generator=_gen(25), device="cuda").bfloat16().repeat(257, 1)[:rows]
    out, part = quantize_float8(x), quantize_float8(x[: 1 << 16])
    assert torch.equal(_bits(out.codes)[: 256 << 16].view(256, 1 << 16, cols), _bits(part.codes).expand(256, -1, -1))
    assert torch.equal(_bits(out.codes)[256 << 16 :], _bits(part.codes)[:5]) and torch.equal(_bits(out.scales)[-5:], _bits(part.scales)[:5])
    weight = torch.linspace(0.5, 2.0, cols, device="cuda").bfloat16()
    (out, h), (part, h_part) = rmsnorm_float8(x, weight, 1e-5, residual=x), rmsnorm_float8(x[: 1 << 16], weight, 1e-5, residual=x[: 1 << 16])
    assert torch.equal(_bits(out.codes)[: 256 << 16].view(256, 1 << 16, cols), _bits(part.codes).expand(256, -1, -1))
    assert torch.equal(_bits(out.codes)[256 << 16 :], _bits(part.codes)[:5]) and torch.equal(_bits(out.scales)[-5:], _bits(part.scales)[:5])
    assert torch.equal(h[-5:], h_part[:5])


# ---- offsets that pass 32 bits -----------------------------------------------------------------------


def _large(rows, cols, seed):
    """Codes of more than 4 GiB (bytes below 0x70: no NaN), and scales around 1."""
    gen = _gen(seed)
    codes = torch.randint(0, 0x70, (rows, cols), generator=gen, device="cuda", dtype=torch.uint8).view(F8)
    return codes


@pytest.mark.parametrize("m", [1, 40, 300])
def test_a_weight_of_more_than_4_gib(m):
    n, k = (1 << 21) + 200, 2064
    w = Float8Tensor(_large(n, k, 1), torch.full(((n + 127) // 128, 17), 127, dtype=torch.uint8, device="cuda").view(E8), 128)
    x = quantize_float8(_randn(_gen(11), m, k))
    y = float8_linear(x, w)
    for lo in (0, 1 << 20, n - 300):
        part = Float8Tensor(w.codes[lo : lo + 300], torch.full((3, 17), 127, dtype=torch.uint8, device="cuda").view(E8), 128)
        _check_16(y[:, lo : lo + 300], *oracle.product(_numbers(x), _numbers(part)))


def test_tokens_of_more_than_4_gib_and_their_results():
    m, k, n = (1 << 21) + 77, 2064, 1100
    x = Float8Tensor(_large(m, k, 2), torch.full((m, 17), 120, dtype=torch.uint8, device="cuda").view(E8))
    w = _weight(_gen(12), n, k)
    y = float8_linear(x, w)  # 2.3e9 numbers
    act = float8_swiglu(x, w, w)
    for lo in (0, 1 << 20, m - 100):
        part = Float8Tensor(x.codes[lo : lo + 100], x.scales[lo : lo + 100])
        _check_16(y[lo : lo + 100], *oracle.product(_numbers(part), _numbers(w)))
        oracle.check_quantized(act.codes[lo : lo + 100], act.scales[lo : lo + 100], *oracle.swiglu(_numbers(part), _numbers(w), _numbers(w)))


def test_quantizing_and_norming_more_than_2_31_numbers():
    rows, k = (1 << 19) + 5, 4104
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda").normal_(generator=_gen(13))
    got = quantize_float8(x)
    weight = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    normed, _ = rmsnorm_float8(x, weight, 1e-6)
    block = quantize_float8(x, block_rows=128)
    for lo in (0, rows - 133):
        part = x[lo : lo + 133]
        assert _equal(quantize_float8(part), Float8Tensor(got.codes[lo : lo + 133], got.scales[lo : lo + 133]))
        assert _equal(rmsnorm_float8(part, weight, 1e-6)[0], Float8Tensor(normed.codes[lo : lo + 133], normed.scales[lo : lo + 133]))
    lo = rows // 128 * 128
    assert _equal(quantize_float8(x[lo:], block_rows=128), Float8Tensor(block.codes[lo:], block.scales[rows // 128 :], 128))


# ---- the model -----------------------------------------------------------------------------------------


def _model(device, fuse=True):
    torch.manual_seed(0)
    model = DecoderOnlyModel(ModelConfig.tiny(), dtype=torch.bfloat16).eval().to(device)
    quantize_model_float8_(model)
    assert not fuse or fuse_projections_(model) == 4
    return model


def test_a_model_on_the_device_is_the_hosts():
    host, dev = _model("cpu"), _model("cpu").cuda()
    for a, b in zip(host.state_dict().values(), dev.state_dict().values()):  # quantized on the host
        assert torch.equal(a.view(torch.uint8), b.cpu().view(torch.uint8))
    ids, pos = torch.arange(40) % 512, torch.arange(40)
    with torch.no_grad():
        want = host(ids, pos, q_len=40).logits.float()
        got = dev(ids.cuda(), pos.cuda(), q_len=40).logits.float().cpu()
        plain = _model("cpu", fuse=False)(ids, pos, q_len=40).logits.float()
    # Roundings to bf16 that fall apart move a code here and there: no more than the fused and the unfused form of one side
    # differ by, of which the second rounds gate times up to bf16 in front of its codes.
    assert float((got - want).norm()) <= 1.5 * float((plain - want).norm())


@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, torch.int8])
def test_generation_with_captured_steps(cache_dtype):
    model = _model("cuda")
    prompts = (torch.arange(24, device="cuda") * 7 % 512).view(3, 8)
    eager = GreedyGenerator(model, cache_dtype=cache_dtype, use_graph=False).generate(prompts, 8)
    graph = GreedyGenerator(model, cache_dtype=cache_dtype).generate(prompts, 8)
    assert torch.equal(eager.tokens, graph.tokens) and torch.equal(eager.prefill_logits, graph.prefill_logits)
