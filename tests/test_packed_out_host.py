"""The ``out`` of packed attention: where it may lie. The launch is replaced, so nothing runs on a device."""

from __future__ import annotations

import itertools
import types

import pytest
import torch

from llmopt.kernels import ops

CU = torch.tensor([0, 6], dtype=torch.int32)


def _elements(t):
    """The storage elements of a tensor."""
    return {t.storage_offset() + sum(i * s for i, s in zip(at, t.stride())) for at in itertools.product(*(range(n) for n in t.shape))}


@pytest.fixture
def launched(monkeypatch):
    """The out pointer, token and head stride of each launch."""
    calls = []

    def packed(*args):
        calls.append(args[18:21])
        return 0

    monkeypatch.setattr(ops, "load_library", lambda: types.SimpleNamespace(llmopt_packed_attention=packed))
    monkeypatch.setattr(ops, "_stream_handle", lambda device: None)
    return calls


def test_out_that_shares_memory_with_an_input_is_written_after_the_kernel(launched):
    q, k, v = (torch.randn(6, 2, 64).half() for _ in range(3))
    for out in (q, k, v):
        ops.packed_attention(q, k, v, CU, 0.125, out=out)
        assert not any(t.data_ptr() <= launched[-1][0] < t.data_ptr() + 2 * t.numel() for t in (q, k, v))
    ops.packed_attention(q, k, v, CU, 0.125, out=torch.empty_like(q))
    own = torch.empty_like(q)
    ops.packed_attention(q, k, v, CU, 0.125, out=own)
    assert launched[-1] == (own.data_ptr(), 128, 64)
    # A slice of the projections' own buffer: beside the inputs' rows it is written in place, across them not.
    fused = torch.randn(6, 8, 64).half()
    parts = [fused[:, i : i + 2] for i in (0, 2, 4, 6)]
    ops.packed_attention(*parts[:3], CU, 0.125, out=parts[3])
    assert launched[-1] == (parts[3].data_ptr(), 512, 64)
    ops.packed_attention(*parts[:3], CU, 0.125, out=fused[:, 3:5])
    assert not fused.data_ptr() <= launched[-1][0] < fused.data_ptr() + 2 * fused.numel()


def test_what_may_share_memory():
    flat = torch.zeros(4000)
    views = [flat[o:].as_strided((3, 2, 4), s) for o in (0, 4, 8, 12, 1000) for s in ((8, 4, 1), (32, 4, 1), (32, 8, 2), (4, 12, 1), (40, 4, 1), (0, 4, 1))]
    agree = 0
    for a, b in itertools.product(views, views):
        share = bool(_elements(a) & _elements(b))
        may = ops._may_share_memory(a, b)
        assert may or not share
        agree += may == share
    assert agree > 0.8 * len(views) ** 2  # it may say so of rows that only pass each other
    assert not ops._may_share_memory(flat[:0].view(0, 2, 4), views[0])


def test_out_in_any_order_of_its_dimensions(launched):
    """Only an out whose own elements share memory is refused, whichever of its strides is the inner one."""
    q, k = torch.zeros(6, 4, 64).half(), torch.zeros(6, 2, 64).half()
    flat = torch.zeros(4 * 6 * 4 * 64).half()
    for strides in ((256, 1, 4), (1, 384, 6), (64, 384, 1), (512, 128, 2), (1, 6, 24), (256, 64, 1)):
        out = flat.as_strided((6, 4, 64), strides)
        assert len(_elements(out)) == out.numel()
        assert ops.packed_attention(q, k, k, CU, 0.125, out=out) is out
    launched.clear()
    for strides in ((256, 64, 2), (256, 1, 1), (128, 1, 2), (0, 1, 4), (1, 1, 8)):
        out = flat.as_strided((6, 4, 64), strides)
        assert len(_elements(out)) < out.numel()
        with pytest.raises(ValueError, match="overlap"):
            ops.packed_attention(q, k, k, CU, 0.125, out=out)
    assert not launched
    one = flat.as_strided((1, 4, 64), (0, 64, 1))  # a stride that nothing steps along
    ops.packed_attention(q[:1], k[:1], k[:1], CU, 0.125, out=one)
