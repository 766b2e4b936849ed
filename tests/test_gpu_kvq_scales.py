"""The 8-bit cache under scales of the caller's that are no powers of two (``from_tensors``): every kernel reads code x
scale, and writes keep or outgrow such a scale as the host does.

Bounds: as in test_gpu_kvq.py, and for the tile kernel, which rounds code x scale to bf16 (half a step is 2^-8): a key moves
its score by at most d = 2^-8 of sum |q k| scale, so a weight by at most e^2d - 1 of itself, and a value its part by 2^-8."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from test_gpu_kvq import FORMATS, HALF_P, _each, _filled, _same, _twin

from oracle import kvq_oracle as ko

pytestmark = pytest.mark.gpu

FACTORS = torch.tensor([0.75, 1.3, 1.0, 1 - 2.0**-24, 1 + 2.0**-23, 1.99, 1.5])


def _uneven(scales, seed):
    at = torch.randint(0, len(FACTORS), scales.shape, generator=torch.Generator().manual_seed(seed))
    scales.mul_(FACTORS[at].to(scales.device))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("q_len,block,hd", [(1, 16, 128), (3, 5, 64), (40, 16, 64), (70, 32, 128)])
def test_attention(fmt, dtype, q_len, block, hd):
    heads, kvh = 8, 2
    cache, table = _filled(2, 200, block, kvh, hd, FORMATS[fmt], seed=q_len, spread=0.0)
    _uneven(cache.key_scales, 1)
    _uneven(cache.value_scales, 2)
    lens = torch.tensor([200, 77], dtype=torch.int32, device="cuda")
    q = torch.randn(2, heads, q_len, hd, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(dtype)
    scale = hd**-0.5
    outs = [out.double().cpu().numpy() for out in _each(q, cache, table, lens, scale)]
    keys, values, _ = (t.double().cpu().numpy() for t in cache.gather(0, table, lens))
    u, step = HALF_P[dtype], torch.finfo(dtype).eps / 2
    for s in range(2):
        visible = np.arange(keys.shape[1])[None, :] <= (int(lens[s]) - q_len + np.arange(q_len))[:, None]
        for h in range(heads):
            want, spread, noise = ko.attention(q[s, h].double().cpu().numpy(), keys[s, :, h // 4], values[s, :, h // 4], visible, scale)
            fp32 = ((hd + 8) * 2.0**-24 * noise + 2.0**-20)[:, None]
            for i, got in enumerate(outs):
                rounded = 0.0 if i == 1 else np.expm1(2 * 2.0**-8 * noise)[:, None] + 2.0**-8  # i = 1: the 16-row kernel
                bound = (2 * (u + fp32) + rounded) * spread + step * np.abs(want) + 2.0**-25
                assert np.max(np.abs(got[s, h] - want) / bound) <= 1.0, (i, s, h)


@pytest.mark.parametrize("fmt", FORMATS)
def test_writes(fmt):
    host, dev = _twin(6, 16, 2, 64, FORMATS[fmt], fill=5)
    for caches in ((host.key_scales, dev.key_scales), (host.value_scales, dev.value_scales)):
        for t in caches:
            _uneven(t, 4)
    table = torch.arange(6, dtype=torch.int32).view(3, 2)
    gen = torch.Generator().manual_seed(6)
    for off, gain in ((3, 0.1), (20, 50.0), (5, 300.0)):
        x = torch.randn(3, 2, 64, generator=gen) * gain
        offsets = torch.full((3,), off, dtype=torch.int32)
        host.write_decode(1, table, offsets, x, -x)
        dev.write_decode(1, table.cuda(), offsets.cuda(), x.cuda(), -x.cuda())
        _same(host, dev)
