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


def _attend(q, cache, table, lens, algo, workspace, nbytes):
    """The C entry point, with a workspace of the caller's."""
    seqs, heads, q_len, hd = q.shape
    q = q.contiguous()
    out = torch.full((seqs, heads, q_len, hd), float("nan"), dtype=q.dtype, device="cuda")
    codes, scales, value_codes, value_scales = cache.layer(0)
    _lib.call(
        _lib.load_library().llmopt_kvq_attention(
            q.data_ptr(), DTYPE_CODES[q.dtype], *q.stride()[:3], codes.data_ptr(), scales.data_ptr(), value_codes.data_ptr(),
            value_scales.data_ptr(), KVQ_FORMATS[cache.dtype], cache.num_blocks, cache.block_size, cache.num_kv_heads, hd,
            table.data_ptr(), int(table.shape[1]), lens.data_ptr(), seqs, heads, q_len, hd**-0.5, 0.0, out.data_ptr(),
            *out.stride()[:3], algo, workspace, nbytes, torch.cuda.current_stream().cuda_stream),
        "llmopt_kvq_attention")
    return out


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("algo,q_len,dtype", [(KVQ_ALGO_ROWS, 1, torch.bfloat16), (KVQ_ALGO_ROWS, 3, torch.float32),
                                              (KVQ_ALGO_TILES, 70, torch.bfloat16), (KVQ_ALGO_TILES, 70, torch.float16)])
def test_without_the_workspace_that_the_splits_ask_for(fmt, algo, q_len, dtype):
    """None, one byte short and off 16 bytes: the context is not split, and the result is the attention all the same."""
    cache, table = _filled(2, 2100, 16, 2, 64, fmt, seed=4)
    lens = torch.tensor([2100, 701], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, q_len, 64, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(dtype)
    need = _lib.load_library().llmopt_kvq_attention_workspace(2, 4, 2, 64, q_len, table.shape[1], 16, DTYPE_CODES[dtype], algo)
    assert need > 0
    space = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    at = space.data_ptr()
    whole = [_attend(q, cache, table, lens, algo, p, n) for p, n in ((None, 0), (None, need), (at, need - 1), (at + 4, need), (at, 0))]
    assert all(torch.equal(w, whole[0]) for w in whole)
    split = _attend(q, cache, table, lens, algo, at, need)
    assert torch.equal(split, ops.kvq_attention(q, *cache.layer(0), table, lens, 0.125, 0.0, algo))
    _check([whole[0], split], q, cache, table, lens, 0.125)


@pytest.mark.parametrize("q_len", [1, 2])
def test_more_splits_than_a_wave_has_lanes(q_len):
    """One KV head and some 33000 tokens are 128 splits; shorter sequences of the batch use some of them, or none."""
    heads, kvh, hd = 4, 1, 64
    lens = torch.tensor([33000, 20000, 16385, 100, 1, 0], dtype=torch.int32, device="cuda")
    for batch in ([0], [1], [2], [3], [0, 4], [2, 5]):
        cache, table = _filled(len(batch), 33000, 16, kvh, hd, torch.int8, seed=6, spread=0.5)
        need = _lib.load_library().llmopt_kvq_attention_workspace(len(batch), heads, kvh, hd, q_len, table.shape[1], 16, 2, 0)
        assert need // (len(batch) * heads * q_len * (hd + 1) * 4) > 64
        q = torch.randn(len(batch), heads, q_len, hd, device="cuda").bfloat16()
        _check(_each(q, cache, table, lens[batch], hd**-0.5), q, cache, table, lens[batch], hd**-0.5)


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_computed_once_more_in_a_split(fmt, dtype):
    """A chunk whose keys are cut into splits, the last of which holds a block marked NaN: queries before that block do not
    see it, and are computed once more within that split."""
    cache, table = _filled(1, 2200, 16, 2, 64, fmt, seed=7)
    lens = torch.tensor([2200], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 8, 100, 64, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda").to(dtype)
    assert _lib.load_library().llmopt_kvq_attention_workspace(1, 8, 2, 64, 100, table.shape[1], 16, DTYPE_CODES[dtype], KVQ_ALGO_TILES) > 0
    cache.value_scales[0, int(table[0, 135])] = float("nan")  # tokens 2160 ..: queries 60 ..
    outs = _each(q, cache, table, lens, 0.125)
    for got in outs:
        assert bool(got[:, :, 60:].isnan().all()) and bool(got[:, :, :60].isfinite().all())
    # what they see: the context in front of the block, as the last tokens of a shorter one
    _check([o[:, :, :60] for o in outs], q[:, :, :60], cache, table, lens - 40, 0.125)
