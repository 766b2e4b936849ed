"""CPU oracle of the 8-bit KV cache and of attention over packed prompts. TEST INFRASTRUCTURE ONLY.

In numpy and float64, written from the definitions and apart from the package's torch and HIP code:

* ``write_tokens`` -- the quantizing write of one sequence's tokens into one layer;
* ``attention`` -- softmax attention of one sequence's query rows over given keys and values with a visibility
  mask, and with it the sums that the tests' error bounds need.
"""

from __future__ import annotations

import math

import numpy as np

TOP = {"int8": 127.0, "e4m3": 448.0}


def scale_for(amax: float, fmt: str) -> float:
    """The smallest 2^e, e >= -126, with amax <= top 2^e; 0 for 0, NaN for what is not finite."""
    if not math.isfinite(amax):
        return math.nan
    if amax == 0:
        return 0.0
    e = -126
    while amax > TOP[fmt] * 2.0**e:
        e += 1
    return 2.0**e


def encode(v: np.ndarray, fmt: str) -> np.ndarray:
    """The format's nearest number, ties to even (np.round's rule)."""
    v = np.asarray(v, dtype=np.float64)
    if fmt == "int8":
        return np.round(v)
    with np.errstate(divide="ignore"):
        exponent = np.floor(np.log2(np.maximum(np.abs(v), 2.0**-6)))
    step = 2.0 ** (exponent - 3)
    return np.round(v / step) * step


def write_tokens(codes, scales, table, offset, x, fmt):  # noqa: ANN001, ANN201
    """``x [n, kv_heads, head_dim]`` from position ``offset`` through ``table`` (block ids) into ``codes [blocks, kv_heads,
    block_size, head_dim]`` and ``scales [blocks, kv_heads]`` (float64), in place."""
    blocks, heads, block_size, _ = codes.shape
    if offset < 0:
        return
    pos, at = offset, 0
    while at < len(x):
        index, slot = divmod(pos, block_size)
        if index >= len(table) or table[index] < 0:
            return
        n = min(block_size - slot, len(x) - at)
        b = table[index]
        if b < blocks:
            for h in range(heads):
                new = x[at : at + n, h].astype(np.float64)
                scale = scale_for(float(np.max(np.abs(new))) if np.isfinite(new).all() else math.nan, fmt)
                if slot > 0:
                    old = scales[b, h]
                    scale = math.nan if math.isnan(old) or math.isnan(scale) else max(old, scale)
                    if not math.isnan(scale) and scale != old:
                        kept = encode(codes[b, h] * (old / scale), fmt)
                        kept[slot : slot + n] = codes[b, h, slot : slot + n]
                        codes[b, h] = kept
                scales[b, h] = scale
                if math.isnan(scale) or scale == 0:
                    codes[b, h, slot : slot + n] = 0
                else:
                    codes[b, h, slot : slot + n] = encode(new / scale, fmt)
        pos, at = pos + n, at + n


def attention(q, k, v, visible, scale, softcap=0.0):  # noqa: ANN001, ANN201
    """``q [rows, d]``, ``k``/``v`` ``[keys, d]``, ``visible [rows, keys]`` (float64): ``(out, spread, noise)`` -- the
    attention, zeros for a row that sees nothing; ``spread`` the same weights over ``|v|``; ``noise [rows]`` the
    largest sum of ``|q k| scale`` over a row's keys, what a score's fp32 rounding errors are relative to."""
    q, k, v = (np.asarray(t, dtype=np.float64) for t in (q, k, v))
    s = q @ k.T * scale
    if softcap > 0:
        s = np.tanh(s / softcap) * softcap
    s = np.where(visible, s, -np.inf)
    any_key = visible.any(1)
    top = np.where(any_key, s.max(1, initial=-np.inf), 0.0)
    p = np.where(visible, np.exp(s - top[:, None]), 0.0)
    total = p.sum(1)
    w = p / np.where(total > 0, total, 1.0)[:, None]
    seen = visible.any(0)
    v0 = np.where(seen[:, None], v, 0.0)
    noise = np.where(visible, np.abs(q) @ np.abs(k).T * abs(scale), 0.0).max(1, initial=0.0)
    return w @ v0, w @ np.abs(v0), noise
