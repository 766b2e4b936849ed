"""Packed attention into a given ``out``: the same bits as without one, wherever it lies."""

from __future__ import annotations

import pytest
import torch

from llmopt.attention import PackedAttention

pytestmark = pytest.mark.gpu


def _same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_out_is_an_input(which, dtype):
    gen = torch.Generator(device="cuda").manual_seed(4)
    qkv = [torch.randn(700, 4, 64, generator=gen, device="cuda").to(dtype) for _ in range(3)]
    qkv[2][90, 1, 5] = float("nan")  # rows that are computed once more, from the query
    cu = torch.tensor([0, 600, 690], dtype=torch.int32, device="cuda")
    attention = PackedAttention(4, 4, 64)
    want, before = attention.forward(*qkv, cu), qkv[which].clone()
    assert attention.forward(*qkv, cu, out=qkv[which]) is qkv[which]
    assert _same(qkv[which][:690], want[:690]) and _same(qkv[which][690:], before[690:])


@pytest.mark.parametrize("at", [6, 5, 3, 0])
def test_out_lies_in_the_projections_own_buffer(at):
    gen = torch.Generator(device="cuda").manual_seed(5)
    fused = torch.randn(300, 8, 128, generator=gen, device="cuda").bfloat16()
    parts = [fused[:, :2], fused[:, 2:4], fused[:, 4:6]]
    cu = torch.tensor([0, 200, 300], dtype=torch.int32, device="cuda")
    attention = PackedAttention(2, 2, 128)
    want = fused.clone()
    want[:, at : at + 2] = attention.forward(*parts, cu)
    attention.forward(*parts, cu, out=fused[:, at : at + 2])
    assert torch.equal(fused, want)
