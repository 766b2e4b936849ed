"""The 8-bit KV cache on the GPU: the writes' codes and scales against the host class (checked number for number against
the oracle in test_kvq_host.py), and PagedAttention over the cache against the float64 oracle.

Bounds of the attention, per output: with u the half step of a probability (2^-8 where it is rounded to bf16, 2^-16 where
it is held in two pieces) the weights p (1 + u) / sum p (1 + u) move an output by at most 2 u sum w |v|; a score's fp32
rounding errors, at most (d + 8) 2^-24 of sum |q k| scale plus 2^-20 for the exponential, move it by twice that times sum w |v|; and
the output is rounded once, by half its type's step."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from llmopt.attention import PagedAttention, PagedAttentionConfig
from llmopt.cache import PagedKVCache, QuantizedPagedKVCache
from llmopt.kernels import ops
from llmopt.kernels._lib import KVQ_ALGO_ROWS, KVQ_ALGO_TILES
from llmopt.model import GreedyGenerator, ModelConfig, random_quantized_model
from oracle import kvq_oracle as ko

pytestmark = pytest.mark.gpu

FORMATS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
HALF_P = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-16, torch.float32: 2.0**-16}


def _twin(blocks, block, heads, hd, dtype, fill=0):
    """The same cache on the host and on the GPU, with earlier contents if `fill`."""
    host = QuantizedPagedKVCache(2, blocks, block, heads, hd, dtype=dtype)
    if fill:
        gen = torch.Generator().manual_seed(fill)
        for codes, scales in ((host.key_codes, host.key_scales), (host.value_codes, host.value_scales)):
            codes.copy_((torch.randn(codes.shape, generator=gen) * 40).round().clamp(-127, 127).to(dtype))
            scales.copy_(torch.exp2(torch.randint(-9, 1, scales.shape, generator=gen).float()))
    return host, QuantizedPagedKVCache.from_tensors(*(t.cuda() for t in (host.key_codes, host.key_scales, host.value_codes,
                                                                        host.value_scales)))


def _same(host, dev):
    for a, b in zip((host.key_codes, host.value_codes, host.key_scales, host.value_scales),
                    (dev.key_codes, dev.value_codes, dev.key_scales, dev.value_scales)):
        a, b = a.float(), b.cpu().float()
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a.nan_to_num(), b.nan_to_num())


# ---- writes ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("block,heads,hd", [(16, 8, 128), (32, 4, 64), (8, 3, 128), (1, 2, 64), (5, 3, 20), (64, 1, 128), (7, 2, 257)])
def test_writes_match_the_host(fmt, dtype, block, heads, hd):
    gen = torch.Generator().manual_seed(block + hd)
    blocks, seqs = 4 * (-(-100 // block)) + 3, 4
    host, dev = _twin(blocks, block, heads, hd, FORMATS[fmt], fill=11)
    width = blocks // seqs
    table = torch.randperm(blocks, generator=gen)[: seqs * width].view(seqs, width).to(torch.int32)
    pos = torch.tensor([0, 3, 0, 1], dtype=torch.int32)
    for step, n in enumerate([37, 1, 1, 18, 1, 5]):
        k = (torch.randn(seqs, n, heads, hd, generator=gen) * 3.0 ** (step % 4)).to(dtype)
        v = (torch.randn(seqs, n, heads, hd, generator=gen) * 0.02 * 5.0 ** (step % 3)).to(dtype)
        if n == 1:
            host.write_decode(1, table, pos, k[:, 0], v[:, 0])
            dev.write_decode(1, table.cuda(), pos.cuda(), k[:, 0].cuda(), v[:, 0].cuda())
        elif step == 3:
            lens = torch.tensor([n, 0, n - 5, 1], dtype=torch.int32)
            host.write(1, table, pos, k, v, query_lens=lens)
            dev.write(1, table.cuda(), pos.cuda(), k.cuda(), v.cuda(), query_lens=lens.cuda())
        else:
            # packed, from views with other strides, rows behind the last sequence not numbers
            lens = torch.tensor([n, 2, n - 1, 0])
            cu = torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(lens, 0)]).to(torch.int32)
            rows = [torch.cat([t[s, : lens[s]] for s in range(seqs)]) for t in (k, v)]
            rows = [torch.cat([t, torch.full((3, heads, hd), float("nan"), dtype=dtype)]) for t in rows]
            host.write_packed(1, table, pos, cu, *rows)
            both = torch.cat(rows, dim=1).cuda()  # [tokens, 2 heads, hd]
            dev.write_packed(1, table.cuda(), pos.cuda(), cu.cuda(), both[:, :heads], both[:, heads:])
        _same(host, dev)
        pos = pos + n


@pytest.mark.parametrize("fmt", FORMATS)
def test_write_borders(fmt):
    """Scales at the ends of the range, ties, subnormal codes, zeros, infinities and NaN."""
    top = ko.TOP[fmt]
    rows = [top, top * (1 + 2**-20), -top / 2, 1e-45, 2.0**-149, 3.4e38, 2.0**-126 * top, 0.0, 1.0, float("inf"), float("nan"), -float("inf")]
    host, dev = _twin(len(rows) + 1, 16, 2, 64, FORMATS[fmt])
    x = torch.zeros(len(rows), 16, 2, 64)
    x[:, 0, 0, 0] = torch.tensor(rows)
    x[:, 1:, 0] = torch.linspace(-1, 1, 15 * 64).view(15, 64) * torch.tensor(rows)[:, None, None].nan_to_num(1, 1, 1)
    x[8, 1, 1] = (torch.arange(64) - 32) / 2 / 64  # halves of a step
    table = torch.arange(len(rows), dtype=torch.int32)[:, None]
    off = torch.zeros(len(rows), dtype=torch.int32)
    for cache in (host, dev):
        d = cache.device
        cache.write(0, table.to(d), off.to(d), x.to(d), -x.to(d))
        grow = torch.full((len(rows), 2, 64), 1.0).to(d) * torch.tensor([1e-3, 1.0, 1e30, 1e-44] * 3)[:, None, None].to(d)
        cache.write_decode(0, table.to(d), (off + 7).to(d), grow, grow)
    _same(host, dev)


def test_write_of_padding_missing_blocks_and_nothing():
    host, dev = _twin(6, 16, 2, 64, torch.int8, fill=3)
    table = torch.tensor([[-1, 2], [9, -1], [1, -1], [0, 7]], dtype=torch.int32)
    one = torch.full((4, 2, 64), 100.0)
    for offsets in ([1, 2, -3, 20], [32, 16, 5, 17], [-1, -1, -1, -1]):
        off = torch.tensor(offsets, dtype=torch.int32)
        host.write_decode(0, table, off, one, one)
        dev.write_decode(0, table.cuda(), off.cuda(), one.cuda(), one.cuda())
        _same(host, dev)
    rows = torch.randn(4, 40, 2, 64)
    off = torch.tensor([0, 3, 15, 16], dtype=torch.int32)
    host.write(0, table, off, rows, rows)
    dev.write(0, table.cuda(), off.cuda(), rows.cuda(), rows.cuda())
    _same(host, dev)
    for cu, n in (([0], 4), ([0, 0, 0, 0, 0], 4), ([0, 0, 0, 0, 0], 0)):
        x = torch.full((n, 2, 64), float("nan"))
        dev.write_packed(0, table.cuda(), off.cuda(), torch.tensor(cu).cuda(), x.cuda(), x.cuda())
    _same(host, dev)


def test_packed_write_of_many_sequences():
    """More sequences than a wave has lanes, most of them short, some empty."""
    gen = torch.Generator().manual_seed(2)
    seqs, heads, hd, block = 5000, 1, 64, 16
    lens = torch.randint(0, 4, (seqs,), generator=gen)
    lens[77] = 250
    cu = torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(lens, 0)]).to(torch.int32)
    off = torch.randint(0, 3, (seqs,), generator=gen).to(torch.int32) * 16
    table = torch.full((seqs, 19), -1, dtype=torch.int32)
    table[:, 0], table[:, 1], table[:, 2] = torch.arange(seqs), torch.arange(seqs) + seqs, torch.arange(seqs) + 2 * seqs
    table[77, 3:] = torch.arange(16) + 3 * seqs
    host, dev = _twin(3 * seqs + 16, block, heads, hd, torch.int8)
    x = torch.randn(int(cu[-1]), heads, hd, generator=gen)
    host.write_packed(0, table, off, cu, x, -x)
    dev.write_packed(0, table.cuda(), off.cuda(), cu.cuda(), x.cuda(), -x.cuda())
    _same(host, dev)


# ---- attention -------------------------------------------------------------------------------------


def _filled(seqs, longest, block, kvh, hd, dtype, seed, spread=1.0):
    """A cache whose blocks hold random codes under scales a factor `spread` apart, its table in no order."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    width = -(-longest // block)
    blocks = seqs * width + 2
    shape = (1, blocks, kvh, block, hd)
    parts = []
    for _ in range(2):
        codes = torch.randn(shape, generator=gen, device="cuda") * 50
        codes = (codes.round() if dtype == torch.int8 else codes).clamp(-127, 127).to(dtype)
        scales = torch.exp2(torch.round(torch.randn(shape[:3], generator=gen, device="cuda") * spread) - 6)
        parts += [codes, scales]
    table = torch.randperm(blocks, generator=gen, device="cuda")[: seqs * width].view(seqs, width).to(torch.int32)
    return QuantizedPagedKVCache.from_tensors(*parts), table


def _check(outs, q, cache, table, lens, scale, softcap=0.0):
    """Each of `outs` against the oracle over what the cache holds, within the bounds of this module's docstring."""
    seqs, heads, q_len, hd = q.shape
    group = heads // cache.num_kv_heads
    keys, values, valid = (t.cpu() for t in cache.gather(0, table, lens))
    u, step = HALF_P[q.dtype], torch.finfo(q.dtype).eps / 2
    outs = [out.double().cpu().numpy() for out in outs]
    assert all(np.isfinite(got).all() for got in outs)
    for s in range(seqs):
        ctx = int(lens[s])
        t = np.arange(keys.shape[1])
        visible = (t[None, :] <= (ctx - q_len + np.arange(q_len))[:, None]) & valid[s].numpy()[None, :]
        for h in range(heads):
            want, spread, noise = ko.attention(q[s, h].double().cpu().numpy(), keys[s, :, h // group].double().numpy(),
                                               values[s, :, h // group].double().numpy(), visible, scale, softcap)
            fp32 = ((hd + 8) * 2.0**-24 * noise + 2.0**-20)[:, None]
            bound = 2 * (u + fp32) * spread + step * np.abs(want) + 1e-30
            if q.dtype == torch.float16:
                bound = bound + 2.0**-25  # half a step of the smallest fp16 numbers
            for i, got in enumerate(outs):
                worst = np.max(np.abs(got[s, h] - want) / bound)
                assert worst <= 1.0, (i, s, h, worst)


def _each(q, cache, table, lens, scale, softcap=0.0):
    """The attention by PagedAttention and by every kernel that takes the query: [(output)]."""
    attention = PagedAttention(q.shape[1], cache.num_kv_heads, q.shape[3], scale=scale, config=PagedAttentionConfig(softcap=softcap))
    outs = [attention.forward(q, cache, 0, table, lens)]
    for algo in (KVQ_ALGO_ROWS, KVQ_ALGO_TILES)[: 1 if q.dtype == torch.float32 else 2]:
        outs.append(ops.kvq_attention(q, *cache.layer(0), table, lens, scale, softcap, algo))
    for out in outs:
        assert out.dtype == q.dtype and out.shape == q.shape
    return outs


SHAPES = [  # seqs, heads, kv_heads, head_dim, block, lengths
    (1, 32, 8, 128, 16, [641]),
    (3, 32, 8, 128, 16, [1, 17, 333]),
    (4, 32, 4, 64, 32, [64, 63, 65, 2000]),
    (2, 6, 2, 64, 16, [100, 31]),
    (2, 5, 5, 128, 8, [77, 40]),
    (3, 16, 1, 128, 5, [1, 64, 129]),
    (2, 40, 2, 64, 1, [33, 70]),
    (2, 7, 1, 128, 48, [500, 47]),
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_decode_attention(fmt, dtype, shape):
    seqs, heads, kvh, hd, block, lens = shape
    cache, table = _filled(seqs, max(lens), block, kvh, hd, FORMATS[fmt], seed=hd + block)
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(seqs, heads, 1, hd, device="cuda").to(dtype)
    _check(_each(q, cache, table, lens, hd**-0.5), q, cache, table, lens, hd**-0.5)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("q_len,shape", [(2, SHAPES[1]), (5, SHAPES[2]), (33, SHAPES[2]), (65, SHAPES[3]), (100, SHAPES[0]), (64, SHAPES[5]),
                                         (40, SHAPES[4]), (130, SHAPES[7]), (9, SHAPES[6])])
def test_chunk_attention(fmt, dtype, q_len, shape):
    seqs, heads, kvh, hd, block, lens = shape
    longest = max(max(lens), q_len)
    cache, table = _filled(seqs, longest, block, kvh, hd, FORMATS[fmt], seed=q_len)
    lens = torch.tensor([max(n, q_len) for n in lens], dtype=torch.int32, device="cuda")
    # token-major rows of a wider tensor: strides that are not contiguous
    wide = torch.randn(seqs, q_len, heads + 1, hd, device="cuda").to(dtype)
    q = wide[:, :, :heads].permute(0, 2, 1, 3)
    _check(_each(q, cache, table, lens, hd**-0.5), q, cache, table, lens, hd**-0.5)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("seqs,heads,kvh,hd,block,q_len,longest", [(4, 32, 8, 128, 16, 200, 900), (1, 32, 8, 128, 16, 300, 3000),
                                                                  (2, 24, 8, 64, 48, 700, 2500), (3, 5, 5, 128, 7, 1100, 1500)])
def test_chunks_that_the_rule_gives_to_the_tile_kernel(fmt, dtype, seqs, heads, kvh, hd, block, q_len, longest):
    """Whole and split over the keys; the same numbers as when the kernel is asked for."""
    cache, table = _filled(seqs, longest, block, kvh, hd, FORMATS[fmt], seed=q_len)
    lens = torch.tensor([longest - 31 * s for s in range(seqs)], dtype=torch.int32, device="cuda")
    q = torch.randn(seqs, q_len, heads, hd, device="cuda").to(dtype).permute(0, 2, 1, 3)
    auto, _, tiles = _each(q, cache, table, lens, hd**-0.5)
    assert torch.equal(auto, tiles)
    some = torch.tensor([0, heads // kvh], device="cuda")  # a head of the first and of the second KV head
    part = QuantizedPagedKVCache.from_tensors(*(t[:, :, :2].contiguous() for t in (cache.key_codes, cache.key_scales, cache.value_codes,
                                                                                  cache.value_scales)))
    _check([auto[:, some]], q[:, some], part, table, lens, hd**-0.5)


@pytest.mark.parametrize("q_len", [1, 3, 70])
def test_rows_without_keys_and_missing_blocks(q_len):
    heads, kvh, hd, block = 8, 2, 64, 16
    cache, table = _filled(6, 160, block, kvh, hd, torch.int8, seed=4)
    table[0, 1], table[1, 0], table[2, :], table[3, 2] = -1, -1, -1, 10**6
    lens = torch.tensor([100, 100, 100, 100, 0, max(0, q_len - 2)], dtype=torch.int32, device="cuda")
    q = torch.randn(6, heads, q_len, hd, device="cuda").bfloat16()
    outs = _each(q, cache, table, lens, hd**-0.5)
    _check(outs, q, cache, table, lens, hd**-0.5)
    for out in outs:
        assert not bool(out[2].any()) and not bool(out[4].any())
        if q_len > 2:
            assert not bool(out[5, :, :2].any()) and bool(out[5, :, 2:].any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kvh,hd", [(71, 1, 64), (131, 1, 128), (600, 2, 64)])
def test_wide_groups(dtype, heads, kvh, hd):
    cache, table = _filled(2, 70, 16, kvh, hd, torch.int8, seed=11)
    lens = torch.tensor([70, 5], dtype=torch.int32, device="cuda")
    q = torch.randn(2, heads, 3, hd, generator=torch.Generator(device="cuda").manual_seed(12), device="cuda").to(dtype)
    _check(_each(q, cache, table, lens, hd**-0.5), q, cache, table, lens, hd**-0.5)


@pytest.mark.parametrize("q_len", [1, 3, 70])
def test_a_table_without_columns(q_len):
    cache, _ = _filled(2, 50, 16, 2, 64, torch.int8, seed=2)
    table = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    lens = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    for out in _each(torch.ones(2, 4, q_len, 64, dtype=torch.bfloat16, device="cuda"), cache, table, lens, 0.1):
        assert not bool(out.any())


@pytest.mark.parametrize("q_len", [1, 4, 80])
@pytest.mark.parametrize("scale,softcap", [(0.3, 5.0), (-0.1, 0.0), (0.0, 0.0)])
def test_scale_and_softcap(q_len, scale, softcap):
    cache, table = _filled(2, 150, 16, 2, 128, torch.float8_e4m3fn, seed=6, spread=0.5)
    lens = torch.tensor([150, 81], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, q_len, 128, device="cuda").bfloat16()
    for dtype in (torch.bfloat16, torch.float16):
        _check(_each(q.to(dtype), cache, table, lens, scale, softcap), q.to(dtype), cache, table, lens, scale, softcap)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("scale,softcap", [(0.5, 64.0), (0.5, 65.0), (-0.3, 1e5), (0.5, 0.25)])
def test_soft_caps_of_both_kinds(dtype, scale, softcap):
    cache, table = _filled(2, 150, 16, 2, 64, torch.int8, seed=13)
    lens = torch.tensor([150, 40], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 33, 64, generator=torch.Generator(device="cuda").manual_seed(14), device="cuda").to(dtype)
    _check(_each(q, cache, table, lens, scale, softcap), q, cache, table, lens, scale, softcap)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_len", [1, 48])
def test_scales_far_apart(fmt, dtype, q_len):
    """Blocks whose scales are up to 2^34 apart: neither a probability nor a product may vanish or overflow."""
    cache, table = _filled(2, 300, 16, 2, 64, FORMATS[fmt], seed=9, spread=0.0)
    cache.value_scales.copy_(torch.exp2(torch.randint(-30, 4, cache.value_scales.shape, device="cuda").float()))
    cache.value_scales[0, table[0].long()] = 2.0**-30  # a sequence of nothing but small values
    lens = torch.tensor([300, 290], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 8, q_len, 64, device="cuda").to(dtype)
    _check(_each(q, cache, table, lens, 0.125), q, cache, table, lens, 0.125)


@pytest.mark.parametrize("q_len", [1, 6, 70])
def test_what_lies_behind_the_context_does_not_matter(q_len):
    cache, table = _filled(3, 200, 16, 2, 128, torch.float8_e4m3fn, seed=12)
    lens = torch.tensor([100, 97, 128], dtype=torch.int32, device="cuda")
    q = torch.randn(3, 8, q_len, 128, device="cuda").bfloat16()
    want = _each(q, cache, table, lens, 0.1)
    for s in range(3):
        first = -(-int(lens[s]) // 16)
        later = table[s, first:].long()
        for scales in (cache.key_scales, cache.value_scales):
            scales[0, later] = float("nan")
        block, slot = int(table[s, int(lens[s]) // 16]), int(lens[s]) % 16
        for codes in (cache.key_codes, cache.value_codes):
            codes.view(torch.uint8)[0, later] = 0x7F
            if slot:
                codes.view(torch.uint8)[0, block, :, slot:] = 0x7F  # NaN codes of another request
    for a, b in zip(_each(q, cache, table, lens, 0.1), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_later_block_that_is_not_finite_leaves_earlier_queries_alone(fmt, dtype):
    """A chunk's last tokens are in a block marked NaN: queries before that block do not see it."""
    cache, table = _filled(1, 128, 16, 2, 64, FORMATS[fmt], seed=13)
    lens = torch.tensor([128], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 8, 100, 64, device="cuda").to(dtype)
    want = _each(q, cache, table, lens, 0.125)
    cache.value_scales[0, int(table[0, 7])] = float("nan")
    for got, was in zip(_each(q, cache, table, lens, 0.125), want):
        assert bool(got[:, :, 84:].isnan().all()) and bool(got[:, :, :84].isfinite().all())
        # Where they are computed once more, key by key, it is without the probabilities' rounding to bf16.
        assert float((got[:, :, :84] - was[:, :, :84]).abs().max()) <= 4 * 2.0**-8 * float(was[:, :, :84].abs().max())
    cache.value_scales[0, int(table[0, 7])] = 1.0
    cache.key_scales[0, int(table[0, 7])] = float("nan")
    for got, was in zip(_each(q, cache, table, lens, 0.125), want):
        assert not bool(got[:, :, 84:].any()) and torch.equal(got[:, :, :84], was[:, :, :84])  # no sum: zeros


def test_decode_without_a_workspace_and_at_every_split():
    """The context of one sequence, and of many, cut in every way the batch sizes give."""
    heads, kvh, hd = 32, 8, 128
    for seqs, ctx in ((1, 5000), (2, 4097), (7, 1500), (33, 640), (130, 300)):
        cache, table = _filled(seqs, ctx, 16, kvh, hd, torch.int8, seed=seqs)
        lens = torch.randint(1, ctx + 1, (seqs,), device="cuda", dtype=torch.int32)
        lens[0] = ctx
        q = torch.randn(seqs, heads, 1, hd, device="cuda").bfloat16()
        out = PagedAttention(heads, kvh, hd).forward(q, cache, 0, table, lens)
        some = torch.unique(torch.cat([torch.tensor([0, seqs - 1]), torch.randint(0, seqs, (2,))])).cuda()
        _check([out[some]], q[some], cache, table[some], lens[some], hd**-0.5)


def test_a_cache_past_32_bits():
    """Codes at byte offsets past 2^32: the last blocks of a layer of 5 GB."""
    blocks, kvh, hd, block = 320_000, 8, 128, 16
    cache = QuantizedPagedKVCache(1, blocks, block, kvh, hd, device="cuda")
    assert cache.key_codes.numel() > 1 << 32
    host = QuantizedPagedKVCache(1, 8, block, kvh, hd)
    table = torch.tensor([[blocks - 1, 3, blocks - 5, blocks - 2, 0, blocks // 2, blocks - 3]], dtype=torch.int32, device="cuda")
    local = torch.arange(7, dtype=torch.int32)[None]
    k, v = torch.randn(1, 100, kvh, hd), torch.randn(1, 100, kvh, hd)
    off = torch.zeros(1, dtype=torch.int32)
    cache.write(0, table, off.cuda(), k.cuda(), v.cuda())
    cache.write_decode(0, table, off.cuda() + 100, 9 * k[:, 0].cuda(), 9 * v[:, 0].cuda())
    host.write(0, local, off, k, v)
    host.write_decode(0, local, off + 100, 9 * k[:, 0], 9 * v[:, 0])
    lens = torch.tensor([101], dtype=torch.int32)
    got = cache.gather(0, table, lens.cuda())
    for a, b in zip(got, host.gather(0, local, lens)):
        assert torch.equal(a.cpu(), b)
    for q_len in (1, 40):
        q = torch.randn(1, 32, q_len, hd, device="cuda").bfloat16()
        _check(_each(q, cache, table, lens.cuda(), hd**-0.5), q, cache, table, lens, hd**-0.5)


# ---- as it is used ---------------------------------------------------------------------------------


def test_steps_captured_and_replayed_beside_each_other():
    """Two captured decode steps (append, attention) of two batches, replayed in turn with eager work between."""
    heads, kvh, hd, ctx = 32, 8, 128, 500

    class Batch:
        def __init__(self, seqs, seed):
            self.cache, self.table = _filled(seqs, ctx + 40, 16, kvh, hd, torch.int8, seed)
            self.lens = torch.full((seqs,), ctx, dtype=torch.int32, device="cuda")
            self.q = torch.randn(seqs, heads, 1, hd, device="cuda").bfloat16()
            self.k, self.v = (torch.randn(seqs, kvh, hd, device="cuda").bfloat16() for _ in range(2))
            self.attention = PagedAttention(heads, kvh, hd)

        def step(self):
            self.lens.add_(1)
            self.cache.write_decode(0, self.table, self.lens - 1, self.k * self.lens[:, None, None] / ctx, self.v)
            return self.attention.forward(self.q, self.cache, 0, self.table, self.lens)

    batches = [Batch(3, 1), Batch(5, 2)]
    graphs, outs = [], []
    for b in batches:
        b.step()
        b.lens.fill_(ctx)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            outs.append(b.step())
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(graph)
    twins = [Batch(3, 1), Batch(5, 2)]
    for t, b in zip(twins, batches):
        t.q, t.k, t.v = b.q, b.k, b.v
        t.step()
        t.lens.fill_(ctx)
        b.lens.fill_(ctx)
    for _ in range(20):
        for i in (0, 1):
            graphs[i].replay()
            want = twins[i].step()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want)
    for t, b in zip(twins, batches):
        assert torch.equal(t.cache.key_codes, b.cache.key_codes) and torch.equal(t.cache.value_scales, b.cache.value_scales)


def test_work_on_a_side_stream_keeps_its_order():
    cache, table = _filled(4, 3000, 16, 8, 128, torch.int8, seed=21)
    lens = torch.full((4,), 2500, dtype=torch.int32, device="cuda")
    q = torch.randn(4, 32, 1, 128, device="cuda").bfloat16()
    attention = PagedAttention(32, 8, 128)
    want = attention.forward(q, cache, 0, table, lens).clone()
    side = torch.cuda.Stream()
    for _ in range(5):
        late = torch.zeros_like(q)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            a = torch.randn(3000, 3000, device="cuda")
            late.copy_(q + 0 * (a @ a)[0, 0])
            out = attention.forward(late, cache, 0, table, lens)
        side.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_generation_over_an_8_bit_cache(dtype):
    """The generator over the 8-bit cache: the kernels' path against the torch path on the same model, graphs and all."""
    config = ModelConfig.tiny()
    model = random_quantized_model(config, device="cuda", dtype=torch.bfloat16, seed=3)
    prompts = torch.randint(0, config.vocab_size, (3, 37), generator=torch.Generator().manual_seed(1))
    forced = torch.randint(0, config.vocab_size, (3, 24), generator=torch.Generator().manual_seed(2))
    got = GreedyGenerator(model, cache_dtype=dtype).generate(prompts, 24, forced=forced)
    eager = GreedyGenerator(model, cache_dtype=dtype, use_graph=False).generate(prompts, 24, forced=forced)
    assert torch.equal(got.tokens, eager.tokens) and torch.equal(got.prefill_logits, eager.prefill_logits)
    wide = GreedyGenerator(model).generate(prompts, 24, forced=forced)
    # Keys and values are off by up to 1/127 (int8) or 1/16 (e4m3) of a block's largest: the logits follow at that order.
    limit = 0.05 if dtype == torch.int8 else 0.2
    assert float((got.prefill_logits - wide.prefill_logits).norm() / wide.prefill_logits.norm()) < limit
    assert isinstance(model.allocate_cache(4, 16, dtype, "cuda"), QuantizedPagedKVCache)
    assert isinstance(model.allocate_cache(4, 16, torch.bfloat16, "cuda"), PagedKVCache)


def test_other_head_dims_take_the_torch_sequence():
    cache, table = _filled(2, 50, 16, 2, 96, torch.int8, seed=2)
    lens = torch.tensor([50, 20], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 3, 96, device="cuda")
    with pytest.raises(NotImplementedError):
        ops.kvq_attention(q, *cache.layer(0), table, lens, 0.1)
    _check([PagedAttention(4, 2, 96).forward(q, cache, 0, table, lens)], q, cache, table, lens, 96**-0.5)


def test_refusals_on_the_device():
    cache, table = _filled(2, 50, 16, 2, 64, torch.int8, seed=2)
    lens = torch.tensor([50, 20], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="same device"):
        cache.write_decode(0, table, lens - 1, torch.zeros(2, 2, 64), torch.zeros(2, 2, 64))
    with pytest.raises(RuntimeError, match="same device"):
        ops.kvq_attention(torch.zeros(2, 4, 1, 64), *cache.layer(0), table, lens, 0.1)
    with pytest.raises(ValueError):
        PagedAttention(4, 2, 64).forward(torch.zeros(2, 3, 1, 64, device="cuda").half(), cache, 0, table, lens)


def test_generation_from_prompts_of_different_lengths():
    """Packed prefill, quantized cache and graph-replayed decode steps of a ragged batch, against each prompt alone."""
    config = ModelConfig.tiny()
    model = random_quantized_model(config, device="cuda", dtype=torch.bfloat16, seed=4)
    gen = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, config.vocab_size, (n,), generator=gen) for n in (3, 130, 64, 1)]
    forced = torch.randint(0, config.vocab_size, (4, 20), generator=gen)
    generator = GreedyGenerator(model, cache_dtype=torch.int8)
    together = generator.generate(prompts, 20, forced=forced)
    eager = GreedyGenerator(model, cache_dtype=torch.int8, use_graph=False).generate(prompts, 20, forced=forced)
    assert torch.equal(together.tokens, eager.tokens)
    for s, p in enumerate(prompts):
        alone = generator.generate([p], 20, forced=forced[s : s + 1])
        # bf16 activations through two layers: other kernels for other batch sizes round differently, by 2^-8 a step
        far = (together.prefill_logits[s] - alone.prefill_logits[0]).norm() / alone.prefill_logits[0].norm()
        assert float(far) < 0.03, (s, float(far))


def test_any_form_of_the_metadata_and_without_the_native_path(monkeypatch):
    cache, table = _filled(3, 600, 16, 2, 128, torch.int8, seed=30)
    twin = QuantizedPagedKVCache.from_tensors(*(t.clone() for t in (cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales)))
    lens = torch.tensor([599, 200, 17], dtype=torch.int32, device="cuda")
    q = torch.randn(3, 8, 1, 128, device="cuda").half()
    k, v = torch.randn(3, 2, 128, device="cuda").half(), torch.randn(3, 2, 128, device="cuda").half()
    attention = PagedAttention(8, 2, 128)
    cache.write_decode(0, table, lens, k, v)
    want = attention.forward(q, cache, 0, table, lens + 1)
    wide = torch.cat([table, table], dim=1).to(torch.int64)[:, : table.shape[1]]
    flat = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")
    flat[1:] = q.reshape(-1)
    for native in (True, False):
        if not native:
            monkeypatch.setattr(ops, "load_binding", lambda: None)
        twin.write_decode(0, wide, lens.cpu().long()[:, None], k.double(), v.double())
        assert torch.equal(twin.key_codes, cache.key_codes) and torch.equal(twin.value_scales, cache.value_scales)
        for layer in (0, -1):
            got = attention.forward(flat[1:].view(q.shape), twin, layer, wide, (lens + 1).long()[:, None])
            assert torch.equal(got, want)
        with pytest.raises(IndexError):
            attention.forward(q, twin, 1, table, lens)
