"""Derivatives through packed prompts and through attention over the 8-bit cache on the GPU: the kernels have none, so
calls that need one take the torch sequence, and none loses a term."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from llmopt.attention import PackedAttention

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
