"""Packed prompts through the attention layer, the model and the generator, on the host: the layer's settings, what it
refuses, and agreement with the paths that take prompts of one length. CPU only."""

from __future__ import annotations

import pytest
import torch

from llmopt.attention import PagedAttention, PagedAttentionConfig
from llmopt.model import DecoderOnlyModel, ModelConfig


def _model(seed=0):
    torch.manual_seed(seed)
    return DecoderOnlyModel(ModelConfig.tiny())


@pytest.mark.parametrize("scale,softcap", [(0.5, 0.0), (None, 0.5), (0.5, 0.5)])
def test_packed_prompts_follow_the_layers_attention(scale, softcap):
    """The settings of ``layer.attn`` hold for packed prompts as they do for prompts of one length over a cache."""
    model = _model()
    for layer in model.layers:
        attn = layer.self_attn
        attn.attn = PagedAttention(attn.num_heads, attn.num_kv_heads, attn.head_dim, scale=scale,
                                   config=PagedAttentionConfig(softcap=softcap), backend="sdpa")
        assert layer.self_attn.packed.backend == "sdpa" and layer.self_attn.packed.softcap == softcap
    ids = torch.randint(0, 512, (2, 9))
    positions = torch.arange(9).repeat(2)
    with torch.no_grad():
        packed = model(ids, positions, cu_seqlens=torch.tensor([0, 9, 18])).logits[0]
        cache = model.allocate_cache(2, 16, torch.float32, "cpu")
        uniform = model(ids, positions, cache=cache, block_ids=torch.tensor([[0], [1]]), context_lens=torch.tensor([9, 9]),
                        q_len=9).logits.reshape(18, -1)
    # the same fp32 sums in another order, through two layers
    torch.testing.assert_close(packed, uniform, atol=1e-5, rtol=1e-4)
