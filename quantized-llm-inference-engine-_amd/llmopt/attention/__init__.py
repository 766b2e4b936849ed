"""Attention over the paged KV cache (``src/llmopt/attention``), and over packed prompts."""

from __future__ import annotations

from llmopt.attention.packed_attention import PackedAttention
from llmopt.attention.paged_attention import (
    AttentionBackend,
    PagedAttention,
    PagedAttentionConfig,
    merge_states,
)

__all__ = ["AttentionBackend", "PackedAttention", "PagedAttention", "PagedAttentionConfig", "merge_states"]
