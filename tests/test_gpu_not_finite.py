"""Infinities and NaN in packed prompts and in the 8-bit cache: the kernels against the host's torch sequences (checked
token by token in test_not_finite_host.py)."""

from __future__ import annotations

import pytest
import torch

from llmopt.attention import PackedAttention

pytestmark = pytest.mark.gpu


def _alike(got, want, dtype):
    """Weights rounded to bf16 or fp16 and one rounding of the output, of values of some units; the same numbers missing."""
    got = got.cpu().float()
    want = want.float()
    assert torch.equal(got.isfinite(), want.isfinite())
    step = torch.finfo(dtype).eps
    torch.testing.assert_close(got.nan_to_num(0, 0, 0), want.nan_to_num(0, 0, 0), atol=8 * step, rtol=2 * step)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("side,bad", [(1, float("nan")), (1, -float("inf")), (2, float("nan")), (2, float("inf")), (0, float("nan"))])
def test_packed_prompts(dtype, hd, side, bad):
    gen = torch.Generator().manual_seed(6)
    qkv = [torch.randn(150, h, hd, generator=gen).to(dtype) for h in (8, 2, 2)]
    qkv[side][70, 1, 9] = bad
    cu = torch.tensor([0, 100, 150], dtype=torch.int32)
    attention = PackedAttention(8, 2, hd)
    _alike(attention.forward(*(t.cuda() for t in qkv), cu.cuda()), attention.forward(*qkv, cu), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_token_whose_scores_are_all_minus_infinity(dtype):
    q, k, v = torch.ones(70, 2, 64, dtype=dtype), torch.ones(70, 1, 64, dtype=dtype), torch.ones(70, 1, 64, dtype=dtype)
    k[:66, 0, 0] = -float("inf")
    out = PackedAttention(2, 1, 64).forward(q.cuda(), k.cuda(), v.cuda(), torch.tensor([0, 70], dtype=torch.int32).cuda())
    assert not bool(out[:66].any()) and bool((out[66:] == 1).all())
