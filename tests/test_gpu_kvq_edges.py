"""Attention over the 8-bit cache at the ends of its arguments: lengths, workspaces, splits, and rows computed once more
in a split. Bounds as in test_gpu_kvq.py."""

from __future__ import annotations

import pytest
import torch
from test_gpu_kvq import _check, _each, _filled

from llmopt.kernels import _lib, ops
from llmopt.kernels._lib import DTYPE_CODES, KVQ_ALGO_ROWS, KVQ_ALGO_TILES, KVQ_FORMATS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_len", [1, 3, 70])
def test_the_ends_of_the_lengths(q_len):
    """A negative context is an empty one, down to the least int32; one past the table ends with it."""
    cache, table = _filled(4, 100, 16, 2, 64, torch.int8, seed=3)
    lens = torch.tensor([-(2**31), -1, -q_len, 2**31 - 1], dtype=torch.int32, device="cuda")
    q = torch.randn(4, 4, q_len, 64, device="cuda").bfloat16()
    whole = torch.full_like(lens, table.shape[1] * 16 + q_len)  # every query behind the table's end
    for got, want in zip(_each(q, cache, table, lens, 0.125), _each(q, cache, table, whole, 0.125)):
        assert not bool(got[:3].any())
        assert torch.equal(got[3], want[3]) and bool(got[3].any())
