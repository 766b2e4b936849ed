"""Infinities and NaN in keys and values on the host: they reach the tokens that see them and no others, as in the
kernels. CPU only."""

from __future__ import annotations

import pytest
import torch

from llmopt.attention import PackedAttention, PagedAttention, PagedAttentionConfig
from llmopt.cache import QuantizedPagedKVCache


def _alike(a, b):
    assert torch.equal(a.isnan(), b.isnan())
    torch.testing.assert_close(a, b, equal_nan=True, atol=2e-6, rtol=1e-5)  # fp32 sums of 20 terms in another order


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("side", ["key", "value"])
def test_packed_prompts(side, bad):
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(33, h, 16, generator=gen) for h in (4, 2, 2))
    cu = torch.tensor([0, 20, 33])
    attention = PackedAttention(4, 2, 16)
    want = attention.forward(q, k, v, cu)
    {"key": k, "value": v}[side][12, 1, 3] = bad
    if side == "value" and bad == float("inf"):
        v[15, 1, 3] = -bad  # both infinities: no number for who sees both
    got = attention.forward(q, k, v, cu)
    assert torch.equal(got[20:], want[20:]) and torch.equal(got[:, :2], want[:, :2])
    _alike(got[:12], want[:12])
    for t in range(12, 20):  # each token alone over what it sees
        for h in (2, 3):
            s = (k[: t + 1, 1] @ q[t, h]) * 16**-0.5
            p = torch.softmax(s, 0)
            _alike(got[t, h], (p[:, None] * v[: t + 1, 1]).sum(0))
    if side == "value":
        assert not bool(got[12:20, 2:, 3].isfinite().any())
        assert bool(got[12:20, 2:, torch.arange(16) != 3].isfinite().all())


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("split", [False, True])
def test_a_block_marked_nan_in_the_8_bit_cache(dtype, split):
    """A chunk's last tokens are in a block marked NaN: queries in front of that block do not see it."""
    gen = torch.Generator().manual_seed(2)
    cache = QuantizedPagedKVCache(1, 6, 8, 2, 16, dtype=dtype)
    table, lens = torch.tensor([[3, 1, 5, 0, 2]]), torch.tensor([40])
    k, v = torch.randn(1, 40, 2, 16, generator=gen), torch.randn(1, 40, 2, 16, generator=gen)
    cache.write(0, table, torch.tensor([0]), k, v)
    q = torch.randn(1, 4, 30, 16, generator=gen)
    attention = PagedAttention(4, 2, 16, config=PagedAttentionConfig(split_kv=split, split_size=12))
    want = attention.forward(q, cache, 0, table, lens)
    cache.value_scales[0, 2, 1] = float("nan")  # tokens 32 .., the second KV head: queries 22 ..
    got = attention.forward(q, cache, 0, table, lens)
    assert torch.equal(got[:, :2], want[:, :2]) and bool(got[:, 2:, 22:].isnan().all())
    _alike(got[:, 2:, :22], want[:, 2:, :22])
    cache.value_scales[0, 2, 1] = 1.0
    cache.key_scales[0, 2, 1] = float("nan")  # no sum: zeros
    got = attention.forward(q, cache, 0, table, lens)
    assert not bool(got[:, 2:, 22:].any())
    _alike(got[:, 2:, :22], want[:, 2:, :22])
    rows = attention.forward(q, cache, 0, table, torch.tensor([10]))
    assert not bool(rows[:, :, :20].any()) and bool(rows[:, :, 20:].all())
    far = attention.forward(q, cache, 0, torch.tensor([[-1, -1, -1, -1, 0]]), lens)  # keys only behind three splits
    assert not bool(far[:, :, :22].any()) and bool(far[:, :, 22:].all())


def test_a_token_whose_scores_are_all_minus_infinity():
    q, k, v = torch.ones(5, 2, 8), torch.ones(5, 1, 8), torch.ones(5, 1, 8)
    k[:2, 0, 0] = -float("inf")
    out = PackedAttention(2, 1, 8).forward(q, k, v, torch.tensor([0, 5]))
    assert not bool(out[:2].any()) and bool((out[2:] == 1).all())
