"""QuantizedPagedKVCache and PackedAttention on the host: the writes' codes and scales against the oracle, number for
number, reads through PagedAttention, packed prompts with their gradients, and every refusal of the entry points
that needs no device. CPU only."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from llmopt.attention import PackedAttention, PagedAttention
from llmopt.cache import PagedKVCache, QuantizedPagedKVCache
from llmopt.kernels import _lib, ops
from llmopt.model import DecoderOnlyModel, GreedyGenerator, ModelConfig
from oracle import kvq_oracle as ko

FORMATS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _numbers(cache):
    return [t.double().numpy() for t in cache.layer(0)]


def _oracle_copy(cache):
    return [t.double().numpy().copy() for t in cache.layer(0)]


def _same(cache, want):
    for got, expected in zip(_numbers(cache), want):
        np.testing.assert_array_equal(got, expected)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("block", [1, 5, 16])
def test_writes_match_the_oracle(fmt, block):
    gen = torch.Generator().manual_seed(3)
    heads, hd, blocks = 2, 12, 40
    cache = QuantizedPagedKVCache(1, blocks, block, heads, hd, dtype=FORMATS[fmt])
    want = _oracle_copy(cache)
    table = torch.randperm(blocks, generator=gen)[:39].view(3, 13)
    table[1, 2] = -1
    pos = [0, 0, 0]
    for step in range(6):  # magnitudes that rise and fall: kept scales, grown scales, new blocks
        n = [3, 1, 7, 2, 1, 4][step]
        k = torch.randn(3, n, heads, hd, generator=gen) * 4.0 ** (step % 3)
        v = torch.randn(3, n, heads, hd, generator=gen) * 0.01 * 4.0 ** (step % 4)
        offsets = torch.tensor(pos)
        if n == 1:
            cache.write_decode(0, table, offsets, k[:, 0], v[:, 0])
        elif step == 2:
            cu = torch.tensor([0, n, 2 * n, 3 * n])
            pad = torch.full((2, heads, hd), float("nan"))
            cache.write_packed(0, table, offsets, cu, torch.cat([k.flatten(0, 1), pad]), torch.cat([v.flatten(0, 1), pad]))
        else:
            cache.write(0, table, offsets, k.to(torch.bfloat16), v.to(torch.bfloat16))
            k, v = k.to(torch.bfloat16).float(), v.to(torch.bfloat16).float()
        for s in range(3):
            ko.write_tokens(want[0], want[1], table[s].tolist(), pos[s], k[s].numpy(), fmt)
            ko.write_tokens(want[2], want[3], table[s].tolist(), pos[s], v[s].numpy(), fmt)
            pos[s] += n
        _same(cache, want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_scales_at_the_borders(fmt):
    top = ko.TOP[fmt]
    for amax in (top, top * (1 + 2**-20), top / 2, 1e-45, 2.0**-149, 3.4e38, 2.0**-126 * top, 0.0):
        cache = QuantizedPagedKVCache(1, 1, 4, 1, 2, dtype=FORMATS[fmt])
        x = torch.tensor([[[[amax, -amax / 3]]]], dtype=torch.float32)
        cache.write(0, torch.tensor([[0]]), torch.tensor([0]), x, x)
        scale = float(cache.key_scales[0, 0, 0])
        assert scale == ko.scale_for(float(x[0, 0, 0, 0]), fmt)
        if amax:
            assert math.frexp(scale)[0] == 0.5


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_marks_its_block_until_it_starts_anew(fmt, bad):
    cache = QuantizedPagedKVCache(1, 3, 4, 2, 8, dtype=FORMATS[fmt])
    table = torch.tensor([[0, 1]])
    x = torch.ones(1, 6, 2, 8)
    x[0, 5, 1, 3] = bad
    cache.write(0, table, torch.tensor([0]), x, torch.ones(1, 6, 2, 8))
    assert bool(cache.key_scales[0, 1, 1].isnan()) and bool(cache.key_scales[0, :2, 0].isfinite().all())
    assert bool(cache.value_scales.isfinite().all())
    keys, _, _ = cache.gather(0, table, torch.tensor([6]))
    assert bool(keys[0, 4:, 1].isnan().all()) and bool((keys[0, :, 0] == 1).all()) and bool((keys[0, :4] == 1).all())
    cache.write_decode(0, table, torch.tensor([6]), torch.ones(1, 2, 8), torch.ones(1, 2, 8))
    assert bool(cache.key_scales[0, 1, 1].isnan())
    cache.write(0, table, torch.tensor([4]), torch.ones(1, 1, 2, 8), torch.ones(1, 1, 2, 8))
    assert bool(cache.key_scales[0, 1].isfinite().all())


def test_padding_and_missing_blocks_are_not_written():
    cache = QuantizedPagedKVCache(1, 4, 4, 1, 8)
    cache.key_codes.fill_(7)
    cache.key_scales.fill_(1.0)
    table = torch.tensor([[-1, 2], [9, -1], [1, -1]])
    one = torch.full((3, 1, 8), 100.0)
    cache.write_decode(0, table, torch.tensor([1, 2, -3]), one, one)
    cache.write_decode(0, table, torch.tensor([8, 4, 5]), one, one)  # past the row, and a -1 block
    assert bool((cache.key_codes == 7).all()) and bool((cache.key_scales == 1).all())
    rows = torch.full((3, 3, 1, 8), 1e9)
    rows[2, :2] = 1.0
    cache.write(0, table, torch.tensor([0, 0, 0]), rows, rows, query_lens=torch.tensor([0, -1, 2]))
    assert float(cache.key_scales[0, 1, 0]) == 2.0**-6 and bool((cache.key_codes[0, 1, 0, :2] == 64).all())
    assert bool((cache.key_codes[0, [0, 2, 3]] == 7).all()) and bool((cache.key_codes[0, 1, 0, 2:] == 7).all())


@pytest.mark.parametrize("q_len", [1, 3])
def test_attention_over_the_cache_on_the_host(q_len):
    gen = torch.Generator().manual_seed(5)
    seqs, heads, kvh, hd, block = 3, 4, 2, 16, 4
    cache = QuantizedPagedKVCache(1, 20, block, kvh, hd)
    lens = torch.tensor([9, 17, q_len])
    table = torch.full((seqs, 5), -1)
    order = torch.randperm(20, generator=gen)
    for s in range(seqs):
        n = -(-int(lens[s]) // block)
        table[s, :n] = order[5 * s : 5 * s + n]
    k, v = torch.randn(seqs, 17, kvh, hd, generator=gen), torch.randn(seqs, 17, kvh, hd, generator=gen)
    cache.write(0, table, torch.zeros(seqs, dtype=torch.long), k, v, query_lens=lens)
    q = torch.randn(seqs, heads, q_len, hd, generator=gen)
    out = PagedAttention(heads, kvh, hd).forward(q, cache, 0, table, lens)
    keys, values, _ = cache.gather(0, table, lens)
    # 127 steps for up to twice the block's largest magnitude: half a step is amax / 127 at most.
    for s in range(seqs):
        assert float((keys[s, : lens[s]] - k[s, : lens[s]]).abs().max()) <= float(k.abs().max()) / 127
        for h in range(heads):
            t = np.arange(keys.shape[1])
            visible = t[None, :] <= (int(lens[s]) - q_len + np.arange(q_len))[:, None]
            want, _, _ = ko.attention(q[s, h].numpy(), keys[s, :, h // 2].numpy(), values[s, :, h // 2].numpy(), visible, hd**-0.5)
            np.testing.assert_allclose(out[s, h].numpy(), want, atol=2e-6)  # fp32 sums of 17 terms near 1


def test_cache_of_a_model_and_its_housekeeping():
    model = DecoderOnlyModel(ModelConfig.tiny())
    cache = model.allocate_cache(6, 16, torch.float8_e4m3fn, "cpu")
    assert isinstance(cache, QuantizedPagedKVCache) and isinstance(model.allocate_cache(6, 16, torch.float16, "cpu"), PagedKVCache)
    assert cache.memory_bytes() == 2 * 2 * 6 * 2 * (16 * 64 + 4)
    cache.key_scales.fill_(1.0)
    cache.reset()
    assert not bool(cache.key_scales.any()) and "float8_e4m3fn" in repr(cache)
    ids = torch.arange(10).view(2, 5)
    table = torch.arange(6).view(2, 3)
    with torch.no_grad():
        dense = model(ids, torch.arange(5).repeat(2), cache=model.allocate_cache(6, 16, torch.float32, "cpu"), block_ids=table,
                      context_lens=torch.tensor([5, 5]), q_len=5).logits
        for dtype in (torch.int8, torch.float8_e4m3fn):
            got = model(ids, torch.arange(5).repeat(2), cache=model.allocate_cache(6, 16, dtype, "cpu"), block_ids=table,
                        context_lens=torch.tensor([5, 5]), q_len=5).logits
            assert bool(got.isfinite().all()) and 0 < float((got - dense).norm() / dense.norm()) < 0.1


def _packed(gen, lens, heads, kvh, hd, padding=0):
    total = sum(lens) + padding
    cu = torch.tensor([0, *np.cumsum(lens)], dtype=torch.int32)
    return (torch.randn(total, heads, hd, generator=gen), torch.randn(total, kvh, hd, generator=gen),
            torch.randn(total, kvh, hd, generator=gen), cu)


def test_packed_prompts_on_the_host():
    gen = torch.Generator().manual_seed(7)
    lens, heads, kvh, hd = [5, 0, 1, 12], 6, 2, 24
    q, k, v, cu = _packed(gen, lens, heads, kvh, hd, padding=3)
    for softcap in (0.0, 2.0):
        out = PackedAttention(heads, kvh, hd, softcap=softcap).forward(q, k, v, cu)
        for lo, hi in zip(cu.tolist(), cu.tolist()[1:]):
            n = hi - lo
            for h in range(heads):
                want, _, _ = ko.attention(q[lo:hi, h].numpy(), k[lo:hi, h // 3].numpy(), v[lo:hi, h // 3].numpy(),
                                          np.tril(np.ones((n, n), dtype=bool)), hd**-0.5, softcap)
                np.testing.assert_allclose(out[lo:hi, h].numpy(), want, atol=4e-6)  # fp32 sums of 24 terms of some units
        assert not bool(out[18:].any())
    kept = torch.full_like(q, 9.0)
    assert PackedAttention(heads, kvh, hd).forward(q, k, v, cu, out=kept) is kept
    assert bool((kept[18:] == 9).all()) and not bool((kept[:18] == 9).any())
    nothing = PackedAttention(heads, kvh, hd).forward(q, k, v, torch.tensor([0]))
    assert nothing.shape == q.shape and not bool(nothing.any())


def test_packed_prompts_gradient_on_the_host():
    gen = torch.Generator().manual_seed(8)
    q, k, v, cu = _packed(gen, [3, 4], 2, 1, 4)
    q, k, v = (t.double().requires_grad_() for t in (q, k, v))
    attention = PackedAttention(2, 1, 4)
    # fp32 inside: differences over 1e-2 steps are good to about 1e-4 of values near 1.
    assert torch.autograd.gradcheck(lambda *t: attention.forward(*t, cu), (q, k, v), eps=1e-2, atol=2e-3, rtol=1e-3, nondet_tol=0)
    with pytest.raises(ValueError, match="gradient"):
        attention.forward(q, k, v, cu, out=torch.empty_like(q))


# ---- refusals --------------------------------------------------------------------------------------


def test_cache_constructor_refusals():
    for bad in ((0, 1, 1, 1, 1), (1, 0, 1, 1, 1), (1, 1, 0, 1, 1), (1, 1, 1, 0, 1), (1, 1, 1, 1, 0)):
        with pytest.raises(ValueError):
            QuantizedPagedKVCache(*bad)
    with pytest.raises(TypeError):
        QuantizedPagedKVCache(1, 1, 1, 1, 1, dtype=torch.float16)
    codes, scales = torch.zeros(1, 2, 3, 4, 8, dtype=torch.int8), torch.zeros(1, 2, 3)
    ok = QuantizedPagedKVCache.from_tensors(codes, scales, codes.clone(), scales.clone())
    assert (ok.num_blocks, ok.num_kv_heads, ok.block_size, ok.head_dim) == (2, 3, 4, 8) and ok.key_codes is codes
    for args, error in (((codes[0], scales, codes[0], scales), ValueError), ((codes, scales[0], codes, scales), ValueError),
                        ((codes, scales.double(), codes, scales), ValueError), ((codes.short(), scales, codes, scales), TypeError),
                        ((codes, scales, codes.view(torch.float8_e4m3fn), scales), TypeError),
                        ((codes.transpose(2, 3), scales[:, :, :1].expand(1, 2, 4), codes.transpose(2, 3), scales[:, :, :1].expand(1, 2, 4)), ValueError)):
        with pytest.raises(error):
            QuantizedPagedKVCache.from_tensors(*args)


def test_write_refusals():
    cache = QuantizedPagedKVCache(1, 2, 4, 3, 8)
    table, off = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    good = torch.zeros(2, 1, 3, 8)
    for write in (lambda *a, **k: cache.write(0, *a, **k), lambda *a, **k: ops.kvq_write(*cache.layer(0), *a, **k)):
        for keys, values in ((good, good[:, :, :2]), (good[..., :7], good[..., :7]), (good[0], good[0])):
            with pytest.raises(ValueError):
                write(table, off, keys, values)
        with pytest.raises(TypeError):
            write(table, off, good.int(), good.int())
        with pytest.raises(ValueError):
            write(table[:1], off, good, good)
        with pytest.raises(ValueError):
            write(table, off[:1], good, good)
        with pytest.raises(ValueError):
            write(table, off, good, good, query_lens=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.kvq_write(*cache.layer(0), table, off, good[:, 0], good[:, 0], cu_seqlens=torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.kvq_write(*cache.layer(0), table[0], off, good, good)
    codes, scales = cache.key_codes[0], cache.key_scales[0]
    with pytest.raises(ValueError):
        ops.kvq_write(codes, scales, codes[:1], scales, table, off, good, good)
    with pytest.raises(ValueError):
        ops.kvq_write(codes, scales[:1], codes, scales, table, off, good, good)
    with pytest.raises(TypeError):
        ops.kvq_write(codes.float(), scales, codes.float(), scales, table, off, good, good)
    with pytest.raises(TypeError):
        ops.kvq_write(codes, scales.double(), codes, scales.double(), table, off, good, good)
    with pytest.raises(ValueError):
        ops.kvq_write(codes.transpose(1, 2), scales[:, :1].expand(2, 4), codes.transpose(1, 2), scales[:, :1].expand(2, 4), table, off, good, good)


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn])
def test_a_write_keeps_no_graph(fmt):
    cache = QuantizedPagedKVCache(1, 2, 4, 2, 64, dtype=fmt)
    k = torch.randn(1, 3, 2, 64, requires_grad=True)
    for offset in (1, 1):
        cache.write(0, torch.tensor([[0]]), torch.tensor([offset]), k * 2, k * 3)
    for t in (cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales):
        assert not t.requires_grad


def test_packed_out_whose_rows_overlap_is_refused():
    q, k = torch.zeros(6, 4, 64, dtype=torch.float16), torch.zeros(6, 2, 64, dtype=torch.float16)
    cu = torch.tensor([0, 6], dtype=torch.int32)
    flat = torch.zeros(6 * 4 * 64, dtype=torch.float16)
    for strides in ((0, 64, 1), (256, 0, 1), (128, 64, 1), (64, 128, 1), (256, 32, 1)):
        with pytest.raises(ValueError, match="overlap"):
            ops.packed_attention(q, k, k, cu, 0.125, out=flat.as_strided((6, 4, 64), strides))


def test_attention_refusals():
    cache = QuantizedPagedKVCache(1, 2, 4, 2, 64)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    q = torch.zeros(2, 4, 1, 64)
    for args, error in (((q[0], table, lens), ValueError), ((q[..., :32], table, lens), ValueError), ((q.double(), table, lens), TypeError),
                        ((q, table[0], lens), ValueError), ((q, table[:1], lens), ValueError), ((q, table, lens[:1]), ValueError)):
        with pytest.raises(error):
            ops.kvq_attention(args[0], *cache.layer(0), args[1], args[2], 0.1)
    assert ops.kvq_attention(q[:0], *cache.layer(0), table, lens, 0.1).shape == (0, 4, 1, 64)


def test_packed_refusals():
    with pytest.raises(ValueError):
        PackedAttention(3, 2, 64)
    with pytest.raises(ValueError):
        PackedAttention(2, 2, 0)
    attention = PackedAttention(4, 2, 64)
    q, k = torch.zeros(5, 4, 64), torch.zeros(5, 2, 64)
    cu = torch.tensor([0, 5], dtype=torch.int32)
    for args in ((q[:, :2], k, k, cu), (q, k[:4], k[:4], cu), (q, k, k[:, :1], cu), (q[0], k, k, cu), (q, k, k, cu[None]), (q, k, k, cu[:0])):
        with pytest.raises(ValueError):
            attention.forward(*args)
    with pytest.raises(ValueError):
        attention.forward(q, k, k, cu, out=q[:4])
    half = (q.half(), k.half(), k.half())
    for args, error in (((q, k, k, cu), NotImplementedError), ((half[0], k, k, cu), TypeError),
                        ((half[0][..., :32], half[1][..., :32], half[2][..., :32], cu), NotImplementedError),
                        ((half[0][:, :3], half[1], half[2], cu), ValueError), ((*half, cu[None]), ValueError), ((q.double(), k.double(), k.double(), cu), TypeError)):
        with pytest.raises(error):
            ops.packed_attention(*args, 0.1)
    with pytest.raises(ValueError):
        ops.packed_attention(*half, cu, 0.1, out=q)


def test_c_entry_points_validate_on_the_host():
    lib = _lib.load_library()
    write, attend, packed = lib.llmopt_kvq_write, lib.llmopt_kvq_attention, lib.llmopt_packed_attention

    def kv(fmt=0, nb=4, bs=16, kvh=2, hd=64, ldb=1, seqs=1, q=1, dt=2, ptr=16):
        return write(ptr, ptr, ptr, ptr, fmt, nb, bs, kvh, hd, ptr, ldb, ptr, None, None, ptr, 0, 0, 0, ptr, 0, 0, 0, dt, seqs, q, 0, None)

    assert kv(fmt=2) == -1 and b"format" in lib.llmopt_kvq_last_error()
    assert kv(nb=0) == -1 and kv(bs=0) == -1 and kv(kvh=0) == -1 and kv(hd=0) == -1 and kv(ldb=-1) == -1
    assert kv(dt=3) == -1 and kv(seqs=-1) == -1 and kv(q=-1) == -1 and kv(ptr=None) == -1
    assert kv(nb=1 << 28) == -2 and kv(ldb=1 << 27) == -2 and kv(seqs=1 << 30) == -2 and kv(q=1 << 31) == -2
    assert kv(seqs=0) == 0 and kv(q=0) == 0 and kv(ldb=0) == 0  # nothing to write: no launch

    def at(fmt=0, hd=64, kvh=2, heads=4, seqs=1, q=1, dt=2, ptr=16, codes=16, algo=0, stride=0):
        return attend(ptr, dt, stride, 0, 0, codes, ptr, codes, ptr, fmt, 4, 16, kvh, hd, ptr, 1, ptr, seqs, heads, q, 1.0, 0.0, ptr, 0, 0, 0, algo, None, 0, None)

    assert at(fmt=5) == -1 and at(dt=9) == -1 and at(heads=3) == -1 and at(heads=0) == -1 and at(seqs=-1) == -1 and at(ptr=None) == -1
    assert at(hd=96) == -2 and at(seqs=65536) == -2 and at(q=1 << 30) == -2 and at(codes=24) == -2
    assert at(algo=3) == -1 and at(algo=-1) == -1 and at(algo=2, dt=0) == -2 and at(algo=2, stride=4) == -2
    assert at(seqs=0) == 0 and at(q=0) == 0

    def pk(dt=2, seqs=1, tokens=4, heads=4, kvh=2, hd=64, ptr=16, stride=64):
        return packed(ptr, stride, 64, ptr, stride, 64, ptr, stride, 64, dt, ptr, seqs, tokens, heads, kvh, hd, 1.0, 0.0, ptr, stride, 64, 1, None)

    assert pk(dt=7) == -1 and pk(seqs=-1) == -1 and pk(tokens=-1) == -1 and pk(heads=3) == -1 and pk(ptr=None) == -1
    assert pk(dt=0) == -2 and pk(hd=80) == -2 and pk(ptr=8) == -2 and pk(stride=65) == -2 and pk(stride=1 << 25) == -2 and pk(tokens=1 << 30) == -2
    assert pk(tokens=0) == 0
    assert lib.llmopt_kvq_attention_workspace(1, 32, 8, 128, 1, 512, 16, 2, 0) > 0
    assert lib.llmopt_kvq_attention_workspace(1, 32, 7, 128, 1, 512, 16, 2, 0) == 0 and lib.llmopt_kvq_attention_workspace(0, 32, 8, 128, 1, 512, 16, 2, 0) == 0
    with pytest.raises(NotImplementedError, match="16-byte"):
        _lib.call(at(codes=24), "llmopt_kvq_attention")


# ---- packed prompts in the model --------------------------------------------------------------------


def test_packed_prefill_of_a_model():
    """Packed prompts against each prompt alone without a cache, and what the cache holds afterwards."""
    torch.manual_seed(0)
    model = DecoderOnlyModel(ModelConfig.tiny())
    lens = [7, 1, 20]
    prompts = [torch.randint(0, 512, (n,)) for n in lens]
    cu = torch.tensor([0, *np.cumsum(lens)], dtype=torch.int32)
    positions = torch.cat([torch.arange(n) for n in lens])
    cache = model.allocate_cache(9, 8, torch.int8, "cpu")
    table = torch.arange(9, dtype=torch.int32).view(3, 3)
    with torch.no_grad():
        every = model(torch.cat(prompts), positions, cu_seqlens=cu).logits
        last = model(torch.cat(prompts), positions, cache=cache, block_ids=table, cu_seqlens=cu, last_only=True).logits
        assert every.shape == (1, 28, 512) and last.shape == (3, 1, 512)
        for s, p in enumerate(prompts):
            alone = model(p, torch.arange(lens[s]), q_len=lens[s]).logits[0]
            torch.testing.assert_close(every[0, cu[s] : cu[s + 1]], alone, atol=1e-5, rtol=1e-4)
            torch.testing.assert_close(last[s, 0], alone[-1], atol=1e-5, rtol=1e-4)
            again = model.allocate_cache(9, 8, torch.int8, "cpu")
            model(p, torch.arange(lens[s]), cache=again, block_ids=table[s : s + 1], cu_seqlens=torch.tensor([0, lens[s]]))
            for a, b in zip(cache.gather(1, table[s : s + 1], torch.tensor(lens[s : s + 1])),
                            again.gather(1, table[s : s + 1], torch.tensor(lens[s : s + 1]))):
                assert float((a.float() - b.float()).abs().max()) < 0.05  # a code at most where fp32 sums differ in their last bits
        with pytest.raises(TypeError, match="QuantizedPagedKVCache"):
            model(torch.cat(prompts), positions, cache=model.allocate_cache(9, 8, torch.float32, "cpu"), block_ids=table, cu_seqlens=cu)


def test_generation_from_prompts_of_different_lengths():
    torch.manual_seed(1)
    model = DecoderOnlyModel(ModelConfig.tiny())
    prompts = [torch.randint(0, 512, (n,)) for n in (3, 17, 9)]
    generator = GreedyGenerator(model, block_size=8, cache_dtype=torch.int8)
    together = generator.generate(prompts, 6)
    for s, p in enumerate(prompts):
        alone = generator.generate([p], 6)
        torch.testing.assert_close(together.prefill_logits[s], alone.prefill_logits[0], atol=1e-5, rtol=1e-4)
        assert torch.equal(together.tokens[s], alone.tokens[0])
    for bad in ([], [torch.zeros(0, dtype=torch.long)], [torch.zeros(1, 2, dtype=torch.long)]):
        with pytest.raises(ValueError):
            generator.generate(bad, 2)
    with pytest.raises(TypeError, match="QuantizedPagedKVCache"):
        GreedyGenerator(model).generate(prompts, 2)
