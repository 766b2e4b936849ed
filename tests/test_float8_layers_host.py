"""Layers in 8-bit floating point in a model: what is fused and what is left as it is. No device is needed."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from llmopt.model import DecoderOnlyModel, ModelConfig, fuse_projections_
from llmopt.quantization import Float8Linear, quantize_model_float8_


def _model(change=None):
    """Two layers in 8-bit floating point, of which `change` puts something else into the second."""
    torch.manual_seed(0)
    model = DecoderOnlyModel(ModelConfig.tiny(vocab_size=64), dtype=torch.bfloat16).eval()
    quantize_model_float8_(model)
    if change is not None:
        change(model.layers[1])
    return model


def _other(linear, bias=False, dtype=torch.bfloat16, rows=None):
    """A layer of `linear`'s input width with a bias, another compute type or another number of rows."""
    torch.manual_seed(1)
    return Float8Linear.from_float(nn.Linear(linear.in_features, rows or linear.out_features, bias=bias).to(dtype))


def _logits(model):
    ids, pos = torch.arange(10) % 64, torch.arange(10)
    with torch.no_grad():
        return model(ids, pos, q_len=10).logits


@pytest.mark.parametrize("name", ["gate_proj", "up_proj"])
def test_gate_and_up_with_a_bias_stay_two_layers(name):
    def change(layer):
        setattr(layer.mlp, name, _other(getattr(layer.mlp, name), bias=True))

    model = _model(change)
    assert fuse_projections_(model) == 3
    assert model.layers[0].mlp.takes_float8() and not model.layers[1].mlp.takes_float8()
    got, want = _logits(model), _logits(_model(change))
    # the first layer's gated product is rounded to bf16 on its way to the down projection where it is not fused
    assert float((got - want).float().norm() / want.float().norm()) < 0.05


@pytest.mark.parametrize("names", [["up_proj"], ["q_proj"], ["k_proj"], ["up_proj", "v_proj"]])
def test_layers_of_two_compute_types_are_not_fused(names):
    def change(layer):
        for name in names:
            parent = layer.mlp if name == "up_proj" else layer.self_attn
            setattr(parent, name, _other(getattr(parent, name), dtype=torch.float16))

    model = _model(change)
    assert fuse_projections_(model) == 4 - len(names)
    second = model.layers[1]
    assert (second.mlp.gate_up is None) == ("up_proj" in names)
    assert (second.self_attn.qkv_proj is None) == any(name != "up_proj" for name in names)
    with pytest.raises(RuntimeError, match="same dtype"):  # as for any input of another type than a layer's
        _logits(model)


def test_gate_and_up_of_two_shapes_are_not_fused():
    model = _model(lambda layer: setattr(layer.mlp, "up_proj", _other(layer.mlp.up_proj, rows=1)))
    assert fuse_projections_(model) == 3
    assert isinstance(model.layers[1].mlp.up_proj, Float8Linear)
    assert _logits(model).shape == (1, 10, 64)  # one feature of up for all of gate's


def test_q_k_and_v_of_two_widths_are_not_fused():
    def change(layer):
        layer.self_attn.k_proj = Float8Linear.from_float(nn.Linear(64, layer.self_attn.k_proj.out_features, bias=False).bfloat16())

    model = _model(change)
    assert fuse_projections_(model) == 3 and model.layers[1].self_attn.qkv_proj is None
