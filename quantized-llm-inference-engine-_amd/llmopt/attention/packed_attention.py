"""Causal attention over whole prompts of different lengths, packed one after the other.

A prefill batch of ragged prompts needs no padding to the longest: the tokens of all of them lie in one ``[tokens,
heads, head_dim]`` tensor, and ``cu_seqlens`` says where each begins. On HIP devices one gfx950 kernel
(``llmopt_packed_attention``) takes the whole batch, fp16 or bf16, keys and values read where the projections left
them. It attends over keys and values as they were computed, so a prompt whose cache is held in 8 bits
(:class:`llmopt.cache.QuantizedPagedKVCache`, :meth:`write_packed`) is itself processed without that rounding. The
reference batches prompts of equal length only (``src/llmopt/model/layers.py:145-163``).
"""

from __future__ import annotations

import torch

from llmopt.attention.paged_attention import AttentionBackend, weighted_values
from llmopt.utils.autograd import is_differentiated

__all__ = ["PackedAttention"]


class PackedAttention:
    """Causal attention over packed prompts.

    Args:
        num_heads: Query heads.
        num_kv_heads: Key/value heads (query head ``h`` reads KV head ``h // group``).
        head_dim: Per-head dimension.
        scale: Softmax scale, ``head_dim ** -0.5`` by default.
        softcap: With a positive value, scores become ``tanh(score / softcap) * softcap``.
        backend: ``"auto"``, ``"hip"`` or ``"sdpa"`` (see :class:`AttentionBackend`).
    """

    def __init__(self, num_heads: int, num_kv_heads: int, head_dim: int, scale: float | None = None,
                 softcap: float = 0.0, backend: str = "auto") -> None:
        if num_kv_heads < 1 or num_heads < 1 or num_heads % num_kv_heads != 0:
            raise ValueError("num_heads must be a positive multiple of num_kv_heads")
        if head_dim < 1:
            raise ValueError("head_dim must be >= 1")
        self.num_heads = num_heads
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.group_size = num_heads // num_kv_heads
        self.scale = scale if scale is not None else head_dim**-0.5
        self.softcap = softcap
        self.backend = AttentionBackend.detect(backend)

    def forward(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, cu_seqlens: torch.Tensor,
                out: torch.Tensor | None = None) -> torch.Tensor:
        """``query [tokens, heads, head_dim]``, ``key``/``value`` ``[tokens, kv_heads, head_dim]``; sequence ``s`` is
        rows ``cu_seqlens[s]`` up to ``cu_seqlens[s + 1]``, and each token sees its sequence's tokens up to itself.
        ``cu_seqlens [sequences + 1]`` starts at 0 and does not fall. Returns ``[tokens, heads, head_dim]`` in the
        query's dtype; rows behind the last sequence are zeros, in a given ``out`` left as they were.

        fp32, head dims other than 64 and 128, host tensors, backends other than ``"hip"``, and inputs that need a
        gradient or carry a tangent (the kernel has no derivative) run the same sums in torch, one sequence at a time.
        """
        if tuple(query.shape[1:]) != (self.num_heads, self.head_dim) or query.dim() != 3 \
                or tuple(key.shape) != (query.shape[0], self.num_kv_heads, self.head_dim) or key.shape != value.shape:
            raise ValueError(f"expected query [tokens, {self.num_heads}, {self.head_dim}] and key, value [tokens, "
                             f"{self.num_kv_heads}, {self.head_dim}], got {tuple(query.shape)}, {tuple(key.shape)}, "
                             f"{tuple(value.shape)}")
        grad = is_differentiated(query, key, value)
        if self.backend == "hip" and query.device.type == "cuda" and not grad:
            from llmopt.kernels import ops

            try:
                return ops.packed_attention(query, key, value, cu_seqlens, self.scale, self.softcap, out)
            except NotImplementedError:
                pass  # a type or shape outside the kernel: the torch sequence below
        return self._torch_sequence(query, key, value, cu_seqlens, out, grad)

    def _torch_sequence(self, query, key, value, cu_seqlens, out, grad):  # noqa: ANN001, ANN202
        if out is not None and (grad or out.shape != query.shape or out.dtype != query.dtype):
            raise ValueError(f"out must be {tuple(query.shape)} {query.dtype}, and without a gradient")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
            raise ValueError("cu_seqlens must be [sequences + 1]")
        tokens = int(query.shape[0])
        cu = [min(max(int(c), 0), tokens) for c in cu_seqlens.tolist()]
        parts = [torch.zeros_like(query[: cu[0] if len(cu) > 1 else tokens])]
        finite = bool(value.isfinite().all())  # read once, not in every sequence
        for lo, hi in zip(cu, cu[1:]):
            q = query[lo:hi].transpose(0, 1).float()
            k = key[lo:hi].transpose(0, 1).float().repeat_interleave(self.group_size, 0)
            v = value[lo:hi].transpose(0, 1).float().repeat_interleave(self.group_size, 0).contiguous()
            scores = torch.matmul(q, k.transpose(1, 2).contiguous()) * self.scale
            if self.softcap > 0:
                scores = torch.tanh(scores / self.softcap) * self.softcap
            hidden = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=query.device).triu(1)
            scores = scores.masked_fill(hidden, float("-inf"))
            none = (scores == float("-inf")).all(-1, keepdim=True)  # no weights: zeros, as in the kernel
            probs = torch.softmax(scores.masked_fill(none, 0.0), -1).masked_fill(none, 0.0)
            out_rows = torch.matmul(probs, v) if finite else weighted_values(probs, ~hidden, v)
            parts.append(out_rows.transpose(0, 1).to(query.dtype))
        if out is not None:
            if len(cu) > 1:
                out[cu[0] : cu[-1]] = torch.cat(parts[1:])
            return out
        if len(cu) > 1:
            parts.append(torch.zeros_like(query[cu[-1] :]))
        return torch.cat(parts)

    def __repr__(self) -> str:
        return f"PackedAttention(heads={self.num_heads}, kv_heads={self.num_kv_heads}, head_dim={self.head_dim})"
