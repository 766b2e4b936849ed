"""PackedAttention on the GPU against the float64 oracle.

Bounds, per output: a probability rounded to bf16 (u = 2^-8) or fp16 (u = 2^-11, and 2^-25 for the smallest) moves an
output by at most 2 u sum w |v| (2^-25 per key); a score's fp32 rounding errors, at most (d + 8) 2^-24 of sum |q k| scale plus
2^-20 for the exponential, by twice that times sum w |v|; the output is rounded once, by half its type's step."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from llmopt.attention import PackedAttention
from llmopt.cache import QuantizedPagedKVCache
from llmopt.kernels import ops
from oracle import kvq_oracle as ko

pytestmark = pytest.mark.gpu


def _inputs(lens, heads, kvh, hd, dtype, padding=0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    total = sum(lens) + padding
    cu = torch.tensor([0, *np.cumsum(lens)], dtype=torch.int32, device="cuda")
    # one fused projection's output: rows of q, k and v side by side
    qkv = torch.randn(total, heads + 2 * kvh, hd, generator=gen, device="cuda").to(dtype)
    return qkv[:, :heads], qkv[:, heads : heads + kvh], qkv[:, heads + kvh :], cu


def _check(out, q, k, v, cu, scale, softcap=0.0, heads=None):
    hd, group = q.shape[2], q.shape[1] // k.shape[1]
    dtype = q.dtype
    step = torch.finfo(dtype).eps / 2
    got = out.double().cpu().numpy()
    cu = cu.tolist()
    for lo, hi in zip(cu, cu[1:]):
        n = hi - lo
        if n == 0:
            continue
        for h in range(q.shape[1]) if heads is None else heads:
            want, spread, noise = ko.attention(*(t[lo:hi, i].double().cpu().numpy() for t, i in ((q, h), (k, h // group), (v, h // group))),
                                               np.tril(np.ones((n, n), dtype=bool)), scale, softcap)
            fp32 = ((hd + 8) * 2.0**-24 * noise + 2.0**-20)[:, None]
            u = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-11
            bound = 2 * (u + fp32) * spread + step * np.abs(want)
            if dtype == torch.float16:
                bound = bound + n * 2.0**-25 * float(v.abs().max()) + 2.0**-25
            worst = np.max(np.abs(got[lo:hi, h] - want) / bound)
            assert worst <= 1.0, (lo, h, worst)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kvh,hd", [(32, 8, 128), (16, 4, 64), (32, 4, 64), (6, 2, 128), (5, 5, 64), (40, 2, 64)])
@pytest.mark.parametrize("lens", [[1], [101], [64, 65, 63, 1, 0, 129], [3] * 70, [500, 2]])
def test_packed_attention(dtype, heads, kvh, hd, lens):
    q, k, v, cu = _inputs(lens, heads, kvh, hd, dtype, padding=13, seed=len(lens))
    out = PackedAttention(heads, kvh, hd).forward(q, k, v, cu)
    assert out.shape == q.shape and out.dtype == dtype
    _check(out, q, k, v, cu, hd**-0.5)
    assert not bool(out[sum(lens) :].any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kvh,hd", [(4, 4, 128), (8, 2, 128), (11, 1, 64), (71, 1, 64), (131, 1, 128), (600, 2, 64)])
@pytest.mark.parametrize("lens", [[32, 33, 31, 1], [96, 97, 95, 160]])
def test_last_tiles_and_wide_groups(dtype, heads, kvh, hd, lens):
    q, k, v, cu = _inputs(lens, heads, kvh, hd, dtype, seed=9)
    some = sorted({0, 1, heads // 2 - 1, heads // 2, heads - 1})
    _check(PackedAttention(heads, kvh, hd).forward(q, k, v, cu), q, k, v, cu, hd**-0.5, heads=some)
    first, *_ = heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    out = torch.zeros_like(first)
    assert PackedAttention(heads, kvh, hd).forward(*heads_first, cu, out=out) is out
    _check(out, q, k, v, cu, hd**-0.5, heads=some)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_long_prompt(dtype):
    q, k, v, cu = _inputs([4001, 30], 8, 2, 128, dtype, seed=5)
    _check(PackedAttention(8, 2, 128).forward(q, k, v, cu), q, k, v, cu, 128**-0.5, heads=[0, 5])


@pytest.mark.parametrize("scale,softcap", [(0.3, 5.0), (-0.1, 0.0), (0.0, 0.0)])
def test_scale_and_softcap(scale, softcap):
    q, k, v, cu = _inputs([150, 31], 4, 2, 128, torch.bfloat16, seed=2)
    _check(PackedAttention(4, 2, 128, scale=scale, softcap=softcap).forward(q, k, v, cu), q, k, v, cu, scale, softcap)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale,softcap", [(0.5, 64.0), (0.5, 65.0), (-0.3, 1e5), (0.5, 0.25)])
def test_soft_caps_of_both_kinds(dtype, scale, softcap):
    q, k, v, cu = _inputs([150, 31], 4, 2, 64, dtype, seed=10)
    _check(PackedAttention(4, 2, 64, scale=scale, softcap=softcap).forward(q, k, v, cu), q, k, v, cu, scale, softcap)


def test_rows_behind_the_last_sequence():
    q, k, v, cu = _inputs([50, 20], 8, 2, 64, torch.bfloat16, padding=90, seed=3)
    for t in (q, k, v):
        t[70:] = float("nan")
    attention = PackedAttention(8, 2, 64)
    out = attention.forward(q, k, v, cu)
    assert not bool(out[70:].any())
    kept = torch.full_like(out, 7.0)
    assert attention.forward(q, k, v, cu, out=kept) is kept
    assert torch.equal(kept[:70], out[:70]) and bool((kept[70:] == 7).all())
    wide = torch.full((160, 9, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    attention.forward(q, k, v, cu, out=wide[:, :8])
    assert torch.equal(wide[:70, :8], out[:70]) and bool((wide[70:] == 7).all()) and bool((wide[:, 8] == 7).all())
    assert not bool(attention.forward(q, k, v, cu[:1]).any())
    assert attention.forward(q[:0], k[:0], v[:0], cu[:1]).shape == (0, 8, 64)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_not_finite_reaches_only_who_sees_it(bad):
    q, k, v, cu = _inputs([90, 40], 8, 2, 128, torch.bfloat16, seed=4)
    attention = PackedAttention(8, 2, 128)
    want = attention.forward(q, k, v, cu).clone()
    v[60, 1, 17] = bad
    got = attention.forward(q, k, v, cu)
    assert torch.equal(got[90:], want[90:]) and torch.equal(got[:, :4], want[:, :4])
    hit = got[60:90, 4:, 17]
    assert bool((~hit.isfinite()).all()) and bool(got[:60].isfinite().all())
    rest = torch.ones(128, dtype=torch.bool)
    rest[17] = False
    assert bool(got[60:90][..., rest].isfinite().all())
    _check(got[:60], q[:60], k[:60], v[:60], torch.tensor([0, 60]), 128**-0.5)
    v[60, 1, 17] = 0.0
    k[70, 0] = float("nan")
    got = attention.forward(q, k, v, cu)
    assert bool(got[70:90, :4].isnan().all()) and bool(got[:70].isfinite().all()) and bool(got[90:].isfinite().all())


def test_strides_and_alignments_that_the_kernel_does_not_take():
    q, k, v, cu = _inputs([40, 25], 4, 2, 64, torch.float16, seed=6)
    attention = PackedAttention(4, 2, 64)
    want = attention.forward(q, k, v, cu)

    def odd(t):  # the same values in rows that begin off 16 bytes
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    assert torch.equal(attention.forward(odd(q), odd(k), odd(v), cu), want)
    turned = [t.permute(2, 0, 1).contiguous().permute(1, 2, 0) for t in (q, k, v)]
    assert torch.equal(attention.forward(*turned, cu), want)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(attention.forward(*heads_first, cu.long()), want)
    one_key = k[:, :1].expand(65, 2, 64)
    _check(attention.forward(q, one_key, v, cu), q, one_key, v, cu, 0.125)
    out = odd(torch.zeros(65, 4, 64, dtype=torch.float16, device="cuda"))
    assert attention.forward(q, k, v, cu, out=out) is out and torch.equal(out, want)


def test_other_types_and_gradients_take_the_torch_sequence():
    q, k, v, cu = _inputs([20, 7], 4, 2, 64, torch.float32, padding=2, seed=7)
    attention = PackedAttention(4, 2, 64)
    with pytest.raises(NotImplementedError):
        ops.packed_attention(q, k, v, cu, 0.125)
    plain = attention.forward(q, k, v, cu)
    half = [t.half() for t in (q, k, v)]
    # fp16 inputs: half a step of 2^-11 on each of q, k and v, of scores of some units
    assert float((attention.forward(*half, cu) - plain).abs().max()) < 0.02
    leaf = half[0].clone().requires_grad_()
    attention.forward(leaf, half[1], half[2], cu).sum().backward()
    assert leaf.grad is not None and bool(leaf.grad.isfinite().all())
    with torch.no_grad():
        assert not attention.forward(leaf, half[1], half[2], cu).requires_grad


def test_a_prompt_then_its_cache():
    """As a server runs it: packed prompts attended and quantized, then decode steps and a chunk over the 8-bit cache."""
    from llmopt.attention import PagedAttention

    heads, kvh, hd, block = 32, 8, 128, 16
    lens = [100, 1, 333, 17]
    q, k, v, cu = _inputs(lens, heads, kvh, hd, torch.bfloat16, padding=61, seed=8)
    packed = PackedAttention(heads, kvh, hd).forward(q, k, v, cu)
    width = -(-(max(lens) + 3) // block)
    cache = QuantizedPagedKVCache(1, 4 * width, block, kvh, hd, device="cuda")
    table = torch.randperm(4 * width, device="cuda").view(4, width).to(torch.int32)
    cache.write_packed(0, table, torch.zeros(4, dtype=torch.int32, device="cuda"), cu, k, v)
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    last = (cu[1:] - 1).long()
    again = PagedAttention(heads, kvh, hd).forward(q[last].unsqueeze(2), cache, 0, table, ctx)[:, :, 0]
    # The cache's keys and values are off by 2^-7 of a block's largest; the last rows of the prompts say so.
    assert float((again - packed[last]).abs().max()) < 0.1 and bool(again.isfinite().all())
    chunk = q[100 + 1 : 100 + 1 + 333].transpose(0, 1)[None]
    over_cache = PagedAttention(heads, kvh, hd).forward(chunk, cache, 0, table[2:3], ctx[2:3])
    assert float((over_cache[0].transpose(0, 1) - packed[101:434]).abs().max()) < 0.3


def test_captured_and_replayed():
    q, k, v, cu = _inputs([200, 60, 5], 8, 2, 64, torch.bfloat16, padding=50, seed=9)
    attention = PackedAttention(8, 2, 64)
    attention.forward(q, k, v, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = attention.forward(q, k, v, cu)
    torch.cuda.current_stream().wait_stream(side)
    for split in (100, 7, 265, 0):
        cu[1], cu[2] = split, max(split, 150)
        q.mul_(-1)
        graph.replay()
        want = attention.forward(q, k, v, cu)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_many_sequences():
    lens = [int(x) for x in torch.randint(0, 6, (3000,), generator=torch.Generator().manual_seed(1))]
    q, k, v, cu = _inputs(lens, 4, 1, 64, torch.bfloat16, padding=5, seed=10)
    out = PackedAttention(4, 1, 64).forward(q, k, v, cu)
    _check(out, q, k, v, cu, 0.125, heads=[2])
    assert not bool(out[-5:].any())
