"""Packed prompts through the attention layer, the model and the generator, on the host: the layer's settings, what it
refuses, and agreement with the paths that take prompts of one length. CPU only."""

from __future__ import annotations

import pytest
import torch

from llmopt.attention import PagedAttention, PagedAttentionConfig
from llmopt.cache import QuantizedPagedKVCache
from llmopt.model import DecoderOnlyModel, GreedyGenerator, ModelConfig


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


def test_packed_prompts_behind_cached_tokens_are_refused():
    """Packed prompts attend over their own rows only, so a cached prefix in front of them would be lost."""
    model = _model()
    cache = model.allocate_cache(4, 16, torch.int8, "cpu")
    table = torch.arange(4, dtype=torch.int32).view(2, 2)
    ids, positions, cu = torch.arange(12), torch.arange(6).repeat(2), torch.tensor([0, 6, 12])
    layer, hidden = model.layers[0].self_attn, torch.randn(12, model.config.hidden_size)
    with torch.no_grad():
        for offsets in (torch.tensor([0, 3]), torch.tensor([[4], [0]], dtype=torch.int32)):
            with pytest.raises(ValueError, match="position 0"):
                model(ids, positions, cache=cache, block_ids=table, token_offsets=offsets, cu_seqlens=cu)
            with pytest.raises(ValueError, match="position 0"):
                layer(hidden, positions, cache, table, token_offsets=offsets, cu_seqlens=cu)
        assert not bool(cache.key_codes.any())
        want = model(ids, positions, cache=cache, block_ids=table, cu_seqlens=cu).logits
        codes = cache.key_codes.clone()
        cache.reset()
        # zeros are the default, and a negative offset keeps its sequence out of the cache
        got = model(ids, positions, cache=cache, block_ids=table, token_offsets=torch.tensor([0, -1]), cu_seqlens=cu).logits
        assert torch.equal(got, want) and not bool(cache.key_codes[:, 2:].any())
        model(ids, positions, cache=cache, block_ids=table, token_offsets=torch.zeros(2, dtype=torch.int32), cu_seqlens=cu)
        assert torch.equal(cache.key_codes, codes)
        # without a cache there is nothing in front of them
        assert torch.equal(model(ids, positions, token_offsets=torch.tensor([0, 3]), cu_seqlens=cu).logits, want)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_prompts_of_one_length_in_either_form(dtype):
    """A tensor of prompts and a list of the same prompts are the same prefill over an 8-bit cache."""
    generator = GreedyGenerator(_model(2), block_size=8, cache_dtype=dtype)
    prompts = torch.randint(0, 512, (3, 13))
    a, b = generator.generate(prompts, 5), generator.generate(list(prompts), 5)
    assert torch.equal(a.prefill_logits, b.prefill_logits) and torch.equal(a.tokens, b.tokens)


@pytest.mark.parametrize("q_len", [1, 4])
def test_fewer_query_tokens_than_the_query_holds(q_len):
    """Over the 8-bit cache the first ``query_lens`` tokens count, on the host as on the device."""
    gen = torch.Generator().manual_seed(3)
    cache = QuantizedPagedKVCache(1, 4, 16, 2, 32)
    table, lens = torch.arange(4).view(2, 2), torch.tensor([20, 25])
    k = torch.randn(2, 25, 2, 32, generator=gen)
    cache.write(0, table, torch.zeros(2, dtype=torch.long), k, k.flip(1))
    q = torch.randn(2, 4, 6, 32, generator=gen)
    attention = PagedAttention(4, 2, 32)
    out = attention.forward(q, cache, 0, table, lens, q_len)
    assert torch.equal(out, attention.forward(q[:, :, :q_len].contiguous(), cache, 0, table, lens))


def test_an_attention_or_layer_of_the_callers_own():
    """What is put in place of a layer's attention, or of a layer, need not know packed prompts while there are none."""

    class Attention(torch.nn.Module):
        def forward(self, hidden, positions, cache, block_ids, context_lens, token_offsets, q_len):  # noqa: ANN001, ANN201
            return 2 * hidden

    class Layer(torch.nn.Module):
        def forward_chained(self, hidden, pending, positions, cache=None, block_ids=None, context_lens=None,  # noqa: ANN001, ANN201
                            token_offsets=None, q_len=1, defer_mlp=False):
            return hidden, pending

    model = _model()
    model.layers[0].self_attn, model.layers[1] = Attention(), Layer()
    with torch.no_grad():
        assert model(torch.arange(6), torch.arange(6), q_len=6).logits.shape == (1, 6, 512)


def test_heads_that_are_not_the_attentions():
    """Another number of heads in the query or in the 8-bit cache is refused, before a kernel would group them its own way."""
    cache = QuantizedPagedKVCache(1, 2, 16, 2, 64)
    table, lens = torch.tensor([[0]]), torch.tensor([5])
    for attention, heads in ((PagedAttention(8, 4, 64), 8), (PagedAttention(8, 1, 64), 8), (PagedAttention(8, 2, 64), 4)):
        with pytest.raises(ValueError, match="KV heads"):
            attention.forward(torch.zeros(1, heads, 1, 64), cache, 0, table, lens)
