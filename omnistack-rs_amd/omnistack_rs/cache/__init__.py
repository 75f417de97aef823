"""Page-granular compressed KV cache (the paged cache the reference plans
for its serving loop: MANIFEST.md:211-215, ``page_size`` in config.py:43)."""
from .blocks import PagedBlockAttention, paged_block_attention, select_blocks
from .paged import PagedKVAttention, PagedKVCache, paged_attention
from .tree import PagedTreeAttention, paged_tree_attention, tree_masks

__all__ = ["PagedBlockAttention", "PagedKVAttention", "PagedKVCache", "PagedTreeAttention", "paged_attention",
           "paged_block_attention", "paged_tree_attention", "select_blocks", "tree_masks"]
