"""Derivatives through packed prompts and through attention over the 8-bit cache on the GPU: the kernels have none, so
calls that need one take the torch sequence, and none loses a term."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from llmopt.attention import PackedAttention, PagedAttention
from llmopt.cache import QuantizedPagedKVCache
from llmopt.model import ModelConfig
from llmopt.model.layers import PagedAttentionLayer

pytestmark = pytest.mark.gpu


def _packed(dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, tangent = (torch.randn(29, h, 64, generator=gen, device="cuda").to(dtype) for h in (4, 2, 2, 4))
    return q, k, v, tangent, torch.tensor([0, 20, 29], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("which", [0, 1, 2])
def test_a_tangent_through_packed_prompts(which):
    *qkv, tangent, cu = _packed()
    tangent = tangent[:, : qkv[which].shape[1]].contiguous()
    attention = PackedAttention(4, 2, 64)

    def through(device):
        t = [x.to(device) for x in qkv]
        with forward_ad.dual_level():
            t[which] = forward_ad.make_dual(t[which], tangent.to(device))
            return forward_ad.unpack_dual(attention.forward(*t, cu.to(device)))

    got, want = through("cuda"), through("cpu")
    assert got.tangent is not None
    # the same fp32 sums on the host, each rounded once to bf16: one step apart at most where they round apart
    for a, b in zip(got, want):
        torch.testing.assert_close(a.cpu().float(), b.float(), atol=2.0**-8, rtol=2.0**-7)


@pytest.mark.parametrize("q_len", [1, 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_querys_derivatives_over_the_8_bit_cache(dtype, q_len):
    gen = torch.Generator(device="cuda").manual_seed(2)
    cache = QuantizedPagedKVCache(1, 8, 16, 2, 64, device="cuda")
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lens = torch.tensor([50, 31], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(2, 64, 2, 64, generator=gen, device="cuda") for _ in range(2))
    cache.write(0, table, torch.zeros_like(lens), k, v)
    host = QuantizedPagedKVCache.from_tensors(*(t.cpu() for t in (cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales)))
    q, weight = (torch.randn(2, 4, q_len, 64, generator=gen, device="cuda").to(dtype) for _ in range(2))
    attention = PagedAttention(4, 2, 64)
    plain = attention.forward(q, cache, 0, table, lens)
    assert not plain.requires_grad
    grads, tangents = [], []
    for dev, store in (("cuda", cache), ("cpu", host)):
        leaf = q.detach().to(dev).requires_grad_()
        out = attention.forward(leaf, store, 0, table.to(dev), lens.to(dev))
        (out.float() * weight.to(dev).float()).sum().backward()
        grads.append(leaf.grad.cpu().float())
        with torch.no_grad():
            assert not attention.forward(leaf, store, 0, table.to(dev), lens.to(dev)).requires_grad
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(q.to(dev), weight.to(dev))
            tangents.append(forward_ad.unpack_dual(attention.forward(dual, store, 0, table.to(dev), lens.to(dev))).tangent.cpu().float())
    # fp32 sums of 50 terms of some units, of which bf16 results are rounded once
    atol, rtol = (2.0**-8, 2.0**-7) if dtype == torch.bfloat16 else (1e-5, 1e-4)
    for a, b in (grads, tangents):
        assert bool(b.any())
        torch.testing.assert_close(a, b, atol=atol, rtol=rtol)


@pytest.mark.parametrize("cached", [False, True])
def test_a_gradient_through_a_layers_packed_prompts(cached):
    """Every term of it, those through the rotated queries and keys among them: against the layer without fused steps."""
    torch.manual_seed(3)
    config = ModelConfig.tiny()
    layer = PagedAttentionLayer(config, 0).to("cuda", torch.bfloat16)
    cu = torch.tensor([0, 11, 24], dtype=torch.int32, device="cuda")
    positions = torch.cat([torch.arange(11), torch.arange(13)]).cuda()
    hidden, weight = (torch.randn(24, config.hidden_size, device="cuda").bfloat16() for _ in range(2))
    sides = []
    for fused in (True, False):
        layer.fused_ops = fused
        layer.zero_grad()
        cache = QuantizedPagedKVCache(1, 4, 16, config.num_key_value_heads, config.head_dim, device="cuda") if cached else None
        table = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2) if cached else None
        leaf = hidden.clone().requires_grad_()
        (layer(leaf, positions, cache, table, cu_seqlens=cu) * weight).float().sum().backward()
        sides.append([leaf.grad] + [p.weight.grad for p in (layer.q_proj, layer.k_proj, layer.v_proj, layer.o_proj)])
    for a, b in zip(*sides):
        assert b is not None and bool(b.any())
        assert torch.equal(a, b)  # the same torch operations
    with torch.no_grad():  # and without a gradient the kernels, as before
        layer.fused_ops = True
        assert not layer(hidden, positions, cu_seqlens=cu).requires_grad
