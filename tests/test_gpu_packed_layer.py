"""Packed prompts through the layer and the generator on the GPU: the layer's settings and backend, and prompts of one
length in either form."""

from __future__ import annotations

import pytest
import torch

from llmopt.attention import PagedAttention, PagedAttentionConfig
from llmopt.cache import QuantizedPagedKVCache
from llmopt.kernels import ops
from llmopt.model import GreedyGenerator, ModelConfig, random_quantized_model
from llmopt.model.layers import PagedAttentionLayer

pytestmark = pytest.mark.gpu


def test_a_layers_settings_and_backend(monkeypatch):
    torch.manual_seed(1)
    config = ModelConfig.tiny()
    layer = PagedAttentionLayer(config, 0).to("cuda", torch.bfloat16)
    hidden = torch.randn(40, config.hidden_size, device="cuda").bfloat16()
    positions = torch.arange(20, device="cuda").repeat(2)
    cu = torch.tensor([0, 20, 40], dtype=torch.int32, device="cuda")
    settings = {"scale": 0.4, "config": PagedAttentionConfig(softcap=0.7)}
    outs = []
    with torch.no_grad():
        plain = layer(hidden, positions, cu_seqlens=cu)
        for backend in ("hip", "sdpa"):
            layer.attn = PagedAttention(layer.num_heads, layer.num_kv_heads, layer.head_dim, backend=backend, **settings)
            if backend == "sdpa":
                monkeypatch.setattr(ops, "packed_attention", lambda *a: pytest.fail("the kernel was asked for"))
            outs.append(layer(hidden, positions, cu_seqlens=cu).float())
    # bf16 weights and one bf16 rounding of each output in front of the projection, which adds up 256 of them
    near = float((outs[0] - outs[1]).norm() / outs[1].norm())
    assert near < 2 * 2.0**-8 < 10 * float((outs[1] - plain.float()).norm() / outs[1].norm())


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_prompts_of_one_length_in_either_form(dtype):
    config = ModelConfig.tiny()
    model = random_quantized_model(config, device="cuda", dtype=torch.bfloat16, seed=6)
    assert isinstance(model.allocate_cache(1, 16, dtype, "cuda"), QuantizedPagedKVCache)
    generator = GreedyGenerator(model, cache_dtype=dtype)
    prompts = torch.randint(0, config.vocab_size, (3, 45), generator=torch.Generator().manual_seed(7))
    a, b = generator.generate(prompts, 12), generator.generate(list(prompts), 12)
    assert torch.equal(a.prefill_logits, b.prefill_logits) and torch.equal(a.tokens, b.tokens)
