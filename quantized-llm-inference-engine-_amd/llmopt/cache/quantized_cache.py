"""The paged key/value cache in 8 bits: half the memory and half the reads of a 16-bit one.

Codes (``torch.int8`` or ``torch.float8_e4m3fn``) are held per layer as ``[num_blocks, kv_heads, block_size,
head_dim]`` for keys and for values, with one fp32 scale for each block and KV head; a code stands for ``code *
scale``. Block tables, offsets and lengths are those of :class:`llmopt.cache.PagedKVCache`
(``src/llmopt/cache/paged_cache.py:137-331``); the reference has no quantized cache.

The scales are powers of two: with ``top`` the format's largest number (127 or 448), a block and head whose largest
magnitude is ``amax`` takes ``2^e`` for the smallest ``e >= -126`` with ``amax <= top 2^e`` (0 if all is zero), and a number
``x`` the code ``x / 2^e``, rounded to nearest, ties to even. So a code times its scale is exact in bf16 and fp32 (down to bf16's
smallest number, 2^-133: an e4m3 code may be 2^-9 and a scale 2^-126), and the same numbers give the same codes everywhere;
int8 loses at most one bit of its range to it, e4m3 no precision.

A write that holds a block's slot 0 starts the block anew: its scale is that of the new tokens, and what other slots held
is void (a block that another request gave back needs no clearing). Any other write keeps the larger of the old and the
needed scale; where it grew, the block's other slots are rounded to it. Infinities and NaN have no code: a block and head
that one is written to gets the scale NaN and reads as NaN until it is started anew.

On HIP devices a write is one kernel (``llmopt_kvq_write``); on the host the same rules run in torch.
"""

from __future__ import annotations

import torch

__all__ = ["QuantizedPagedKVCache"]


class QuantizedPagedKVCache:
    """Fixed-capacity paged K/V store in 8 bits, shared by all layers.

    Args:
        num_layers: Decoder layers sharing the store.
        num_blocks: Physical blocks per layer.
        block_size: Tokens per block.
        num_kv_heads: Key/value heads.
        head_dim: Per-head dimension.
        dtype: Code format, ``torch.int8`` or ``torch.float8_e4m3fn``.
        device: Device to allocate on.

    Attributes:
        key_codes, value_codes: ``[num_layers, num_blocks, num_kv_heads, block_size, head_dim]`` of ``dtype``.
        key_scales, value_scales: ``[num_layers, num_blocks, num_kv_heads]`` fp32.
    """

    # format -> (largest number, the exponent p and fraction m of it, m 2^p with m in [0.5, 1))
    FORMATS = {torch.int8: (127.0, 7, 127 / 128), torch.float8_e4m3fn: (448.0, 9, 0.875)}

    def __init__(
        self,
        num_layers: int,
        num_blocks: int,
        block_size: int,
        num_kv_heads: int,
        head_dim: int,
        dtype: torch.dtype = torch.int8,
        device: torch.device | str = "cpu",
    ) -> None:
        if num_layers < 1:
            raise ValueError("num_layers must be >= 1")
        if num_blocks < 1 or block_size < 1:
            raise ValueError("num_blocks and block_size must be >= 1")
        if num_kv_heads < 1 or head_dim < 1:
            raise ValueError("num_kv_heads and head_dim must be >= 1")
        if dtype not in self.FORMATS:
            raise TypeError(f"the 8-bit cache holds int8 or float8_e4m3fn codes, not {dtype}")
        shape = (num_layers, num_blocks, num_kv_heads, block_size, head_dim)
        codes = [torch.zeros(shape, dtype=torch.int8, device=device).view(dtype) for _ in range(2)]
        scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)]
        self._adopt(codes[0], scales[0], codes[1], scales[1], shape)

    def _adopt(self, key_codes, key_scales, value_codes, value_scales, shape) -> None:  # noqa: ANN001
        self.key_codes, self.key_scales = key_codes, key_scales
        self.value_codes, self.value_scales = value_codes, value_scales
        self.num_layers, self.num_blocks, self.num_kv_heads, self.block_size, self.head_dim = shape
        self.dtype = key_codes.dtype
        self.device = key_codes.device

    @classmethod
    def from_tensors(cls, key_codes: torch.Tensor, key_scales: torch.Tensor, value_codes: torch.Tensor,
                     value_scales: torch.Tensor) -> QuantizedPagedKVCache:
        """A cache over tensors that exist already (shapes as the attributes; shared, not copied). The codes must be
        finite and the scales not negative. Scales need not be the powers of two that a write gives: a code stands for
        ``code * scale`` under any, and a write keeps the larger scale; attention of chunks then rounds that to bf16."""
        cache = cls.__new__(cls)
        if key_codes.is_cuda:  # the checks below in native code: 0.6 us instead of 4
            from llmopt.kernels import ops

            shape = ops.cache_shape(key_codes, key_scales, value_codes, value_scales)
            if shape is not None:
                cache._adopt(key_codes, key_scales, value_codes, value_scales, shape)
                return cache
        if key_codes.dim() != 5 or key_codes.shape != value_codes.shape or 0 in key_codes.shape:
            raise ValueError(f"expected two [layers, blocks, kv_heads, block_size, head_dim] code tensors, got "
                             f"{tuple(key_codes.shape)} and {tuple(value_codes.shape)}")
        if key_codes.dtype not in cls.FORMATS or value_codes.dtype != key_codes.dtype:
            raise TypeError(f"the 8-bit cache holds int8 or float8_e4m3fn codes, not {key_codes.dtype}, "
                            f"{value_codes.dtype}")
        shape, device = key_codes.shape[:3], key_codes.device
        if key_scales.shape != shape or value_scales.shape != shape or key_scales.dtype != torch.float32 \
                or value_scales.dtype != torch.float32:
            raise ValueError(f"expected float32 scales {tuple(shape)}, got {tuple(key_scales.shape)} "
                             f"{key_scales.dtype} and {tuple(value_scales.shape)} {value_scales.dtype}")
        tensors = (key_codes, key_scales, value_codes, value_scales)
        if not (key_codes.is_contiguous() and key_scales.is_contiguous() and value_codes.is_contiguous()
                and value_scales.is_contiguous()) or not key_scales.device == value_codes.device \
                == value_scales.device == device:
            raise ValueError("the cache's tensors must be contiguous and on one device")
        cache._adopt(*tensors, key_codes.shape)
        return cache

    def layer(self, layer_idx: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """``(key_codes, key_scales, value_codes, value_scales)`` of one layer."""
        return (self.key_codes[layer_idx], self.key_scales[layer_idx], self.value_codes[layer_idx],
                self.value_scales[layer_idx])

    # ---- writes ---------------------------------------------------------------------------------

    def write(
        self,
        layer_idx: int,
        block_ids: torch.Tensor,
        token_offsets: torch.Tensor,
        keys: torch.Tensor,
        values: torch.Tensor,
        query_lens: torch.Tensor | None = None,
    ) -> None:
        """Quantize ``keys``/``values`` ``[seq, q_len, kv_heads, head_dim]`` from position ``token_offsets[s]``, of
        each sequence the first ``query_lens[s]`` tokens (all without it): tokens behind them are padding that must
        not reach a block's scale.

        A sequence's tokens go block by block through its row of ``block_ids`` (``-1`` padded); writing stops at the
        first negative block or at the end of the row; a block id past the cache and a negative offset write nothing.
        No block may belong to two sequences of one call.
        """
        if keys.dim() != 4 or values.dim() != 4:
            raise ValueError(f"write takes [seq, q_len, kv_heads, head_dim], got {tuple(keys.shape)} and "
                             f"{tuple(values.shape)}")
        self._write(layer_idx, block_ids, token_offsets, keys, values, None, query_lens)

    def write_decode(
        self,
        layer_idx: int,
        block_ids: torch.Tensor,
        token_offsets: torch.Tensor,
        keys: torch.Tensor,
        values: torch.Tensor,
    ) -> None:
        """Quantize one token per sequence, ``keys``/``values`` ``[seq, kv_heads, head_dim]``, at ``token_offsets[s]``.
        A token whose block id is not one of the cache's is not written (:class:`PagedKVCache` puts it into block 0,
        whose scale it would spoil here), so ``-1`` rows pad a batch."""
        if keys.dim() != 3 or values.dim() != 3:
            raise ValueError(f"write_decode takes [seq, kv_heads, head_dim], got {tuple(keys.shape)} and "
                             f"{tuple(values.shape)}")
        self._write(layer_idx, block_ids, token_offsets, keys, values, None, None)

    def write_packed(
        self,
        layer_idx: int,
        block_ids: torch.Tensor,
        token_offsets: torch.Tensor,
        cu_seqlens: torch.Tensor,
        keys: torch.Tensor,
        values: torch.Tensor,
    ) -> None:
        """:meth:`write` of sequences of different lengths packed one after the other: ``keys``/``values`` ``[tokens,
        kv_heads, head_dim]``, sequence ``s`` the rows ``cu_seqlens[s]`` up to ``cu_seqlens[s + 1]`` (``cu_seqlens [seq + 1]``
        starts at 0 and does not fall; rows behind the last sequence are not read)."""
        self._write(layer_idx, block_ids, token_offsets, keys, values, cu_seqlens, None)

    def _write(self, layer_idx, block_ids, token_offsets, keys, values, cu_seqlens, query_lens) -> None:  # noqa: ANN001
        if self.key_codes.device.type == "cuda":
            from llmopt.kernels import ops

            ops.cache_write(self, layer_idx, block_ids, token_offsets, keys, values, cu_seqlens, query_lens)
            return
        if cu_seqlens is None and keys.dim() == 3:
            keys, values = keys.unsqueeze(1), values.unsqueeze(1)
        if keys.shape != values.shape or keys.dim() != (4 if cu_seqlens is None else 3) \
                or tuple(keys.shape[-2:]) != (self.num_kv_heads, self.head_dim):
            raise ValueError(f"keys and values of shape {tuple(keys.shape)} and {tuple(values.shape)} do not match the "
                             f"cache's {self.num_kv_heads} heads of {self.head_dim}")
        if not (keys.is_floating_point() and values.is_floating_point()):
            raise TypeError(f"keys and values must be floating-point, got {keys.dtype}, {values.dtype}")
        keys, values = keys.detach(), values.detach()  # the cache is no part of a graph
        table = block_ids.to("cpu", torch.long).tolist()
        starts = token_offsets.reshape(-1).tolist()
        if cu_seqlens is not None:
            cu = [min(max(int(c), 0), int(keys.shape[0])) for c in cu_seqlens.tolist()]
            rows = [(keys[lo:hi], values[lo:hi]) for lo, hi in zip(cu, cu[1:])]
        else:
            lens = [int(keys.shape[1])] * int(keys.shape[0]) if query_lens is None else query_lens.reshape(-1).tolist()
            if len(lens) < int(keys.shape[0]):
                raise ValueError(f"query_lens has {len(lens)} rows for {int(keys.shape[0])} sequences")
            rows = [(k[: max(0, n)], v[: max(0, n)]) for k, v, n in zip(keys, values, lens)]
        if len(table) < len(rows) or len(starts) < len(rows):
            raise ValueError(f"block_ids and token_offsets need a row for each of {len(rows)} sequences")
        key_codes, key_scales, value_codes, value_scales = self.layer(layer_idx)
        for s, (k, v) in enumerate(rows):
            pos, end, at = starts[s], starts[s] + int(k.shape[0]), 0
            while 0 <= pos < end and pos // self.block_size < len(table[s]) and table[s][pos // self.block_size] >= 0:
                block, slot = table[s][pos // self.block_size], pos % self.block_size
                n = min(self.block_size - slot, end - pos)
                if block < self.num_blocks:
                    self._write_block(key_codes[block], key_scales[block], slot, k[at : at + n])
                    self._write_block(value_codes[block], value_scales[block], slot, v[at : at + n])
                pos, at = pos + n, at + n

    def _write_block(self, codes: torch.Tensor, scales: torch.Tensor, slot: int, x: torch.Tensor) -> None:
        """``x [n, kv_heads, head_dim]`` into slots ``slot ..`` of one block (``codes [kv_heads, block_size, head_dim]``)."""
        x = x.float()
        scale = self._scale_for(x.abs().amax((0, 2)))
        if slot > 0:
            old = scales.clone()
            scale = torch.where(old.isnan() | scale.isnan(), torch.nan, torch.maximum(old, scale))
            grown = scale > old
            if bool(grown.any()):
                kept = self._encode(codes[grown].float() * (old[grown] / scale[grown])[:, None, None])
                codes[grown] = kept
        inv = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))[:, None]
        new = torch.where(scale.isnan()[:, None], torch.zeros_like(x), x * inv)
        codes[:, slot : slot + x.shape[0]] = self._encode(new).transpose(0, 1)
        scales.copy_(scale)

    def _scale_for(self, amax: torch.Tensor) -> torch.Tensor:
        """The scale that numbers of magnitude up to ``amax`` need."""
        _, p_top, m_top = self.FORMATS[self.dtype]
        m, p = torch.frexp(amax)
        e = (p - p_top + (m > m_top).to(p.dtype)).clamp(min=-126, max=127)
        scale = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), torch.zeros_like(amax))
        return torch.where(amax.isfinite(), scale, torch.full_like(amax, torch.nan))

    def _encode(self, x: torch.Tensor) -> torch.Tensor:
        return x.round().to(torch.int8) if self.dtype == torch.int8 else x.to(self.dtype)

    # ---- reads ----------------------------------------------------------------------------------

    def gather(
        self,
        layer_idx: int,
        block_ids: torch.Tensor,
        context_lens: torch.Tensor,
    ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Dense ``(keys, values, valid)`` for a ragged batch, as :meth:`PagedKVCache.gather`: keys/values ``[seq,
        max_len, kv_heads, head_dim]`` dequantized to fp32 and padded with zeros, ``valid[s, t]`` true when ``t <
        context_lens[s]`` and the token's block id names a block."""
        seqs = int(block_ids.shape[0])
        dev = self.key_codes.device
        longest = int(context_lens.max().item()) if seqs else 0
        longest = max(0, min(longest, int(block_ids.shape[1]) * self.block_size))
        pos = torch.arange(longest, device=dev)
        ids = block_ids.to(dev, torch.long)[:, pos // self.block_size]
        valid = (ids >= 0) & (ids < self.num_blocks) & (pos[None, :] < context_lens.reshape(-1).to(dev)[:, None])
        ids = torch.where(valid, ids, torch.zeros_like(ids))
        out = []
        for codes, scales in ((self.key_codes, self.key_scales), (self.value_codes, self.value_scales)):
            bits = codes[layer_idx].view(torch.int8)[ids, :, pos % self.block_size]  # [seq, len, kv_heads, head_dim]
            x = bits.view(self.dtype).float() * scales[layer_idx][ids][..., None]
            out.append(torch.where(valid[:, :, None, None], x, torch.zeros_like(x)))
        return out[0], out[1], valid

    # ---- housekeeping ---------------------------------------------------------------------------

    def memory_bytes(self) -> int:
        return 2 * (self.key_codes.numel() + 4 * self.key_scales.numel())

    def reset(self) -> None:
        for codes, scales in ((self.key_codes, self.key_scales), (self.value_codes, self.value_scales)):
            codes.view(torch.int8).zero_()
            scales.zero_()

    def __repr__(self) -> str:
        return (
            f"QuantizedPagedKVCache(layers={self.num_layers}, blocks={self.num_blocks}, "
            f"block_size={self.block_size}, kv_heads={self.num_kv_heads}, head_dim={self.head_dim}, "
            f"dtype={self.dtype}, bytes={self.memory_bytes()})"
        )
