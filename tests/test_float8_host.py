"""8-bit floating point on the host: the definitions against 64 bits, the layers, derivatives, and what is refused. No device
is needed."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from llmopt.kernels import _lib
from llmopt.model import DecoderOnlyModel, GreedyGenerator, ModelConfig, fuse_projections_
from llmopt.quantization import (Float8Linear, Float8SwiGLU, Float8Tensor, FusedFloat8Linear, float8_linear, float8_swiglu, quantize_float8,
                                 quantize_model_float8_, rmsnorm_float8)
from oracle import float8_oracle as oracle

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _x(rows, k, seed=0, dtype=torch.float32):
    return (torch.randn(rows, k, generator=torch.Generator().manual_seed(seed)) * 2).to(dtype)


def _bits(t):
    return t.view(torch.uint8)


# ---- definitions -----------------------------------------------------------------------------------


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 128), (130, 300), (5, 1040)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize(rows, k, block_rows, dtype):
    x = _x(rows, k, dtype=dtype)
    got = quantize_float8(x, block_rows)
    assert got.codes.dtype == F8 and got.scales.dtype == E8 and got.block_rows == block_rows
    oracle.check_quantized(got.codes, got.scales, x.double(), 0.0, block_rows)
    assert torch.equal(got.dequantize().double(), oracle.numbers(got.codes, got.scales, block_rows))


def test_a_scale_is_the_smallest_that_fits():
    top = torch.ldexp(torch.tensor(448.0), torch.arange(-134, 119))
    x = torch.stack([top, torch.nextafter(top, top * 2), torch.nextafter(top, top / 2)], 1).reshape(-1, 1)
    got = quantize_float8(x)
    assert torch.equal(got.scales.double(), oracle.scales_of(x.double(), 1))
    assert torch.equal(got.dequantize()[::3], x[::3])
    assert _bits(quantize_float8(torch.zeros(1, 5)).scales).item() == 0


def test_what_is_not_finite_reads_as_nan():
    x = _x(3, 400)
    x[0, 3], x[1, 200] = float("inf"), float("nan")
    got = quantize_float8(x).dequantize()
    assert bool(got[0, :128].isnan().all()) and bool(got[1, 128:256].isnan().all())
    assert int(got.isnan().sum()) == 256
    y = float8_linear(quantize_float8(x), quantize_float8(_x(7, 400), 128))
    assert y.isnan().all(1).tolist() == [True, True, False]


@pytest.mark.parametrize("residual", [False, True])
def test_norm(residual):
    x, r, w = _x(5, 300, 1, torch.bfloat16), _x(5, 300, 2, torch.bfloat16), _x(1, 300, 3, torch.bfloat16)[0]
    out, h = rmsnorm_float8(x, w, 1e-5, residual=r if residual else None)
    want = r + x if residual else x
    assert torch.equal(h, want)
    h64 = want.double()
    y = h64 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + 1e-5) * w.double()
    oracle.check_quantized(out.codes, out.scales, y, y.abs() * (300 + 8) * 2.0**-24)  # additions in any order


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (4, 130, 200), (2, 5, 1000)])
def test_products(m, n, k):
    x, gate, up = quantize_float8(_x(m, k)), quantize_float8(_x(n, k, 1), 128), quantize_float8(_x(n, k, 2), 128)
    x64, g64, u64 = oracle.numbers(x.codes, x.scales, 1), oracle.numbers(gate.codes, gate.scales, 128), oracle.numbers(up.codes, up.scales, 128)
    bias = _x(1, n, 3, torch.float16)[0]
    want, off = oracle.product(x64, g64)
    y = float8_linear(x, gate, bias, torch.float16)
    want = want + bias.double()
    assert bool(((y.double() - want).abs() <= off + want.abs() * 2.0**-11 * 1.01).all())
    out = float8_swiglu(x, gate, up)
    oracle.check_quantized(out.codes, out.scales, *oracle.swiglu(x64, g64, u64))


def test_leading_dimensions():
    x = _x(6, 200).view(2, 3, 200)
    got = quantize_float8(x)
    assert got.codes.shape == (2, 3, 200) and got.scales.shape == (2, 3, 2) and got.shape == got.codes.shape
    w = quantize_float8(_x(9, 200, 1), 128)
    assert float8_linear(got, w).shape == (2, 3, 9)
    assert float8_swiglu(got, w, w).scales.shape == (2, 3, 1)
    row = quantize_float8(x[0, 0])
    assert row.scales.shape == (2,) and float8_linear(row, w).shape == (9,)
    out, h = rmsnorm_float8(x.bfloat16(), torch.ones(200).bfloat16(), 1e-5)
    assert out.codes.shape == h.shape == (2, 3, 200)


# ---- layers ----------------------------------------------------------------------------------------


def _linear(k, n, bias=False, seed=0):
    torch.manual_seed(seed)
    return nn.Linear(k, n, bias=bias).bfloat16()


@pytest.mark.parametrize("bias", [False, True])
def test_float8_linear_layer(bias):
    dense = _linear(200, 150, bias)
    layer = Float8Linear.from_float(dense)
    assert layer.compute_dtype == torch.bfloat16 and (layer.out_features, layer.in_features) == (150, 200)
    x = _x(4, 200, 1, torch.bfloat16)
    w = quantize_float8(dense.weight.detach(), block_rows=128)
    y = layer(x)
    assert torch.equal(y, float8_linear(quantize_float8(x), w, dense.bias, torch.bfloat16))
    assert torch.equal(layer(quantize_float8(x)), y) and not y.requires_grad
    # e4m3 with scales per block is some 4 % of a typical number
    ref = dense(x).detach().float()
    assert float((y.float() - ref).norm() / ref.norm()) < 0.08


def test_parts_of_one_layer():
    parts = [Float8Linear.from_float(_linear(200, n, b, i)) for i, (n, b) in enumerate([(256, False), (128, True), (70, False)])]
    one, x = FusedFloat8Linear(parts), _x(3, 200, 1, torch.bfloat16)
    got = one(x)
    assert [g.shape[1] for g in got] == one.out_features == [256, 128, 70]
    for g, p in zip(got, parts):  # a bias of zeros changes -0 to 0 at most
        torch.testing.assert_close(g, p(x), atol=0, rtol=0)
    with pytest.raises(ValueError, match="multiple of 128"):
        FusedFloat8Linear(parts[::-1])
    with pytest.raises(ValueError, match="same in_features"):
        FusedFloat8Linear([parts[0], Float8Linear.from_float(_linear(100, 10))])
    with pytest.raises(ValueError, match="nothing"):
        FusedFloat8Linear([])


def test_swiglu_layer():
    gate, up = (Float8Linear.from_float(_linear(200, 150, seed=i)) for i in (1, 2))
    x = _x(4, 200, 1, torch.bfloat16)
    got = Float8SwiGLU(gate, up)(x)
    want = float8_swiglu(quantize_float8(x), gate.weight_tensor(), up.weight_tensor())
    assert torch.equal(_bits(got.codes), _bits(want.codes)) and torch.equal(_bits(got.scales), _bits(want.scales))
    with pytest.raises(ValueError, match="bias"):
        Float8SwiGLU(gate, Float8Linear.from_float(_linear(200, 150, True)))
    with pytest.raises(ValueError, match="shape"):
        Float8SwiGLU(gate, Float8Linear.from_float(_linear(200, 10)))


def test_module_conversions_keep_codes_and_scales():
    layer = Float8Linear.from_float(_linear(200, 150, True))
    codes, scales = layer.weight_codes, layer.weight_scales
    for convert in (lambda m: m.float(), lambda m: m.half(), lambda m: m.to("cpu", torch.float64)):
        convert(layer)
        assert layer.weight_codes.dtype == F8 and layer.weight_scales.dtype == E8 and layer.bias.dtype == torch.bfloat16
        assert torch.equal(_bits(layer.weight_codes), _bits(codes)) and torch.equal(_bits(layer.weight_scales), _bits(scales))
    other = Float8Linear.from_float(_linear(200, 150, True, 1))
    other.load_state_dict(layer.state_dict())
    x = _x(2, 200, 1, torch.bfloat16)
    assert torch.equal(other(x), layer(x))


def test_quantizing_a_model():
    model = nn.Sequential(nn.Linear(100, 60), nn.ReLU(), nn.Sequential(nn.Linear(60, 30, bias=False))).bfloat16()
    model.add_module("lm_head", nn.Linear(30, 10).bfloat16())
    assert quantize_model_float8_(model) is model
    assert isinstance(model[0], Float8Linear) and isinstance(model[2][0], Float8Linear) and type(model.lm_head) is nn.Linear
    assert model(_x(2, 100, 0, torch.bfloat16)).shape == (2, 10)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        quantize_model_float8_(nn.Sequential(nn.Linear(8, 8)))


# ---- the decoder -----------------------------------------------------------------------------------


def _model(fuse=True, **sizes):
    torch.manual_seed(0)
    config = ModelConfig.tiny(vocab_size=64)
    for name, value in sizes.items():
        setattr(config, name, value)
    model = quantize_model_float8_(DecoderOnlyModel(config, dtype=torch.bfloat16).eval())
    return (model, fuse_projections_(model)) if fuse else model


@pytest.mark.parametrize("sizes,fused", [({}, 4), ({"num_key_value_heads": 1}, 2)])
def test_a_model_in_8_bit_floating_point(sizes, fused):
    """Fused projections take the norms' quantized outputs; unfused ones, the same numbers."""
    model, count = _model(**sizes)
    assert count == fused  # a key projection of 64 rows is not fused
    plain = _model(fuse=False, **sizes)
    ids, pos = torch.arange(10) % 64, torch.arange(10)
    with torch.no_grad():
        got = model(ids, pos, q_len=10).logits
        want = plain(ids, pos, q_len=10).logits
    assert got.shape == (1, 10, 64)
    # unfused, the gated product is rounded to bf16 on its way to the down projection: 2^-9 of it, where both round to e4m3
    assert float((got - want).float().norm() / want.float().norm()) < 0.05
    dense = DecoderOnlyModel(model.config, dtype=torch.bfloat16)
    torch.manual_seed(0)
    assert all(m.takes_float8() for layer in model.layers for m in (layer.self_attn, layer.mlp))
    assert not any(m.takes_float8() for layer in dense.layers for m in (layer.self_attn, layer.mlp))


def test_the_norms_hand_on_quantized_outputs_unless_a_derivative_is_needed():
    model, _ = _model()
    seen = []
    for layer in model.layers:
        for m in (layer.self_attn, layer.mlp):
            m.register_forward_pre_hook(lambda mod, args: seen.append(type(args[0])))
    ids, pos = torch.arange(6), torch.arange(6)
    with torch.no_grad():
        model(ids, pos, q_len=6)
    assert seen == [Float8Tensor] * 4
    seen.clear()
    out = model(ids, pos, q_len=6).logits
    assert seen == [torch.Tensor] * 4
    out.float().sum().backward()
    grads = [model.embed_tokens.weight.grad] + [n.weight.grad for layer in model.layers
                                                for n in (layer.input_layernorm, layer.post_attention_layernorm)]
    assert all(g is not None and bool(g.any()) for g in grads)


def test_generation_with_a_model_in_8_bit_floating_point():
    model, _ = _model()
    prompts = torch.arange(12).view(2, 6)
    tokens = GreedyGenerator(model).generate(prompts, 4).tokens
    assert tokens.shape == (2, 4)
    ragged = GreedyGenerator(model, cache_dtype=torch.int8).generate([prompts[0], prompts[1, :3]], 3).tokens
    assert ragged.shape == (2, 3)


# ---- derivatives -----------------------------------------------------------------------------------


def test_a_gradient_goes_straight_through_the_rounding():
    dense = _linear(200, 150, True)
    layer = Float8Linear.from_float(dense)
    x = _x(4, 200, 1, torch.bfloat16).requires_grad_()
    y = layer(x)
    # fp32 sums in another order, each rounded once to bf16: a step apart at most
    torch.testing.assert_close(y.detach().float(), layer(x.detach()).float(), atol=1e-6, rtol=2.0**-7)
    seed = _x(4, 150, 2, torch.bfloat16)
    y.backward(seed)
    want = seed.double() @ oracle.numbers(layer.weight_codes, layer.weight_scales, 128)
    # fp32 sums of 150 terms of the magnitudes below, then a rounding to bf16
    terms = seed.double().abs() @ oracle.numbers(layer.weight_codes, layer.weight_scales, 128).abs()
    assert bool(((x.grad.double() - want).abs() <= terms * 150 * 2.0**-23 + want.abs() * 2.0**-8 * 1.01).all())
    with torch.no_grad():
        assert not layer(x).requires_grad


def test_a_tangent_goes_straight_through_the_rounding():
    layer = Float8Linear.from_float(_linear(200, 150))
    x, t = _x(4, 200, 1, torch.bfloat16), _x(4, 200, 2, torch.bfloat16)
    with torch.autograd.forward_ad.dual_level():
        y = torch.autograd.forward_ad.unpack_dual(layer(torch.autograd.forward_ad.make_dual(x, t)))
    want = t.double() @ oracle.numbers(layer.weight_codes, layer.weight_scales, 128).t()
    assert float((y.tangent.double() - want).norm() / want.norm()) < 2.0**-8


def test_a_bias_has_its_derivative():
    x, w = quantize_float8(_x(6, 64, 1, torch.float32)), quantize_float8(_x(40, 64, 2, torch.float32), block_rows=128)
    bias = torch.zeros(40, dtype=torch.bfloat16, requires_grad=True)
    float8_linear(x, w, bias).sum().backward()
    assert torch.equal(bias.grad, torch.full((40,), 6.0, dtype=torch.bfloat16))


def test_a_gradient_through_the_gated_product():
    gate, up = (Float8Linear.from_float(_linear(64, 50, seed=i)) for i in (1, 2))
    x = _x(4, 64, 1, torch.bfloat16).requires_grad_()
    out = Float8SwiGLU(gate, up)(x)
    assert isinstance(out, torch.Tensor)
    out.sum().backward()
    assert bool(x.grad.abs().gt(0).any())


def test_a_norms_stream_keeps_its_graph():
    x, r = _x(2, 64, 1, torch.bfloat16).requires_grad_(), _x(2, 64, 2, torch.bfloat16)
    out, h = rmsnorm_float8(x, torch.ones(64).bfloat16(), 1e-5, residual=r)
    assert h.requires_grad and not out.codes.requires_grad
    assert not quantize_float8(x).codes.requires_grad


# ---- refusals --------------------------------------------------------------------------------------


def test_refused_tensors():
    with pytest.raises(TypeError, match="floating-point"):
        quantize_float8(torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(TypeError, match="floating-point"):
        quantize_float8(torch.zeros(2, 3).to(F8))
    with pytest.raises(ValueError, match="at least one dimension"):
        quantize_float8(torch.tensor(1.0))
    with pytest.raises(ValueError, match="1 or 128 rows"):
        quantize_float8(torch.zeros(2, 3), block_rows=64)
    with pytest.raises(ValueError, match="2D weight"):
        quantize_float8(torch.zeros(2, 3, 4), block_rows=128)
    codes = torch.zeros(200, 300).to(F8)
    with pytest.raises(TypeError, match="e8m0"):
        Float8Tensor(codes, torch.ones(200, 3))
    with pytest.raises(TypeError, match="e4m3"):
        Float8Tensor(torch.zeros(200, 300), torch.ones(200, 3).to(E8))
    for shape, rows in (((200, 2), 1), ((2, 3), 1), ((200, 3), 128), ((2, 3), 7)):
        with pytest.raises(ValueError):
            Float8Tensor(codes, torch.ones(shape).to(E8), rows)
    with pytest.raises(ValueError):
        Float8Tensor(codes.view(2, 100, 300), torch.ones(2, 3).to(E8), 128)


def test_refused_norms():
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="weight"):
        rmsnorm_float8(x, torch.ones(65), 1e-5)
    with pytest.raises(ValueError, match="residual"):
        rmsnorm_float8(x, torch.ones(64), 1e-5, residual=torch.zeros(1, 64))
    with pytest.raises(ValueError, match="residual"):
        rmsnorm_float8(x, torch.ones(64), 1e-5, residual=x.bfloat16())


def test_refused_products():
    x, w = quantize_float8(torch.zeros(2, 64)), quantize_float8(torch.zeros(8, 64), 128)
    with pytest.raises(RuntimeError, match="cannot be multiplied"):
        float8_linear(x, quantize_float8(torch.zeros(8, 65), 128))
    with pytest.raises(ValueError, match="block_rows"):
        float8_linear(w, w)
    with pytest.raises(ValueError, match="block_rows"):
        float8_linear(x, x)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        float8_linear(x, w, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="same dtype"):
        float8_linear(x, w, torch.zeros(8))
    with pytest.raises(ValueError, match="bias"):
        float8_linear(x, w, torch.zeros(9).bfloat16())
    with pytest.raises(ValueError, match="different shapes"):
        float8_swiglu(x, w, quantize_float8(torch.zeros(9, 64), 128))
    layer = Float8Linear(w)
    with pytest.raises(RuntimeError, match="same dtype"):
        layer(torch.zeros(2, 64))
    with pytest.raises(ValueError, match="128 x 128"):
        Float8Linear(x)
    with pytest.raises(ValueError, match="bias"):
        Float8Linear(w, torch.zeros(9))


def test_the_c_abi_refuses_before_anything_reaches_a_device():
    lib = _lib.load_library()
    p = 1 << 20  # never read

    def quantize(dtype=2, rows=4, cols=256, block=1, ldx=256, ldc=256, lds=2, x=p):
        return lib.llmopt_f8_quantize(x, ldx, dtype, rows, cols, block, p, ldc, p, lds, None)

    assert quantize(dtype=5) == -1 and b"dtype" in lib.llmopt_f8_last_error()
    assert quantize(block=64) == -1 and b"1 or 128 rows" in lib.llmopt_f8_last_error()
    assert quantize(ldx=255) == -1 and b"x: rows" in lib.llmopt_f8_last_error()
    assert quantize(ldc=255) == -1 and b"codes" in lib.llmopt_f8_last_error()
    assert quantize(lds=1) == -1 and b"scales" in lib.llmopt_f8_last_error()
    assert quantize(x=None) == -1 and b"null" in lib.llmopt_f8_last_error()
    assert quantize(rows=-1) == -1 and b"negative" in lib.llmopt_f8_last_error()
    assert quantize(rows=1 << 31, cols=256) == -2
    assert quantize(rows=0) == 0 and quantize(cols=0) == 0

    def norm(dtype=2, h=p, ldh=256, res=p, weight=p):
        return lib.llmopt_f8_rmsnorm(p, 256, res, 256, h, ldh, weight, p, 256, p, 2, 4, 256, 1e-5, dtype, None)

    assert norm(dtype=7) == -1 and norm(dtype=0) == -2
    assert norm(h=None) == -1 and b"h_out" in lib.llmopt_f8_last_error()
    assert norm(ldh=100) == -1 and norm(weight=None) == -1

    def linear(dtype=2, m=4, n=8, ldx=256, ldw=256, ldxs=2, ldws=2, ldy=8, w=p, y=p):
        return lib.llmopt_f8_linear(p, ldx, p, ldxs, m, 256, w, ldw, p, ldws, None, y, ldy, n, dtype, None, 0, None)

    assert linear(dtype=9) == -1 and linear(dtype=0) == -2
    for bad in ({"ldx": 255}, {"ldw": 200}, {"ldxs": 1}, {"ldws": 1, "n": 200, "ldy": 200}, {"ldy": 7}, {"w": None}, {"y": None}):
        assert linear(**bad) == -1, bad
    assert linear(m=0) == 0 and linear(n=0) == 0

    def swiglu(ldg=256, lds=1, n=8, up=p):
        return lib.llmopt_f8_swiglu(p, 256, p, 2, 4, 256, p, ldg, p, 2, up, 256, p, 2, n, p, 8, p, lds, None, 0, None)

    assert swiglu(ldg=255) == -1 and b"gate" in lib.llmopt_f8_last_error()
    assert swiglu(up=None) == -1 and b"up is null" in lib.llmopt_f8_last_error()
    assert swiglu(lds=0) == -1 and swiglu(n=0) == 0


def test_workspaces():
    """None for sizes that are not split or refused, and never more than the parts of eight."""
    lib = _lib.load_library()
    for m, n, k in ((0, 10, 10), (-1, 10, 10), (10, 0, 10), (10, 10, 0), (1, 4096, 4096), (8192, 4096, 14336), (1 << 40, 5, 5)):
        assert lib.llmopt_f8_linear_workspace(m, n, k) == 0, (m, n, k)
    assert lib.llmopt_f8_linear_workspace(32, 4096, 14336) > 0
    for m in (17, 32, 100, 256, 1000):
        for n in (1, 100, 4096, 28672):
            for k in (16, 1040, 14336):
                ws = lib.llmopt_f8_linear_workspace(m, n, k)
                assert 0 <= ws <= 8 * m * (n + 15) * 4 and ws % (m * 64) == 0
    # the gated product's two sums where few tokens or features make that faster, and else none
    assert lib.llmopt_f8_swiglu_workspace(17, 4096, 4096) == 2 * 17 * 4096 * 4
    assert lib.llmopt_f8_swiglu_workspace(500, 4096, 4096) == 0 and lib.llmopt_f8_swiglu_workspace(0, 8, 8) == 0
    assert lib.llmopt_f8_swiglu_workspace(1 << 40, 8, 8) == 0
    assert lib.llmopt_f8_swiglu_workspace(3, 50, 77) == 2 * 3 * 64 * 4


@pytest.mark.parametrize("rc,kind", [(-1, ValueError), (-2, NotImplementedError), (-4, RuntimeError)])
def test_status_codes_raise_with_this_headers_message(rc, kind):
    lib = _lib.load_library()
    assert lib.llmopt_f8_quantize(1 << 20, 4, 9, 1, 4, 1, 1 << 20, 4, 1 << 20, 1, None) == -1
    with pytest.raises(kind, match="bad dtype code 9"):
        _lib.call(rc, "llmopt_f8_quantize")
