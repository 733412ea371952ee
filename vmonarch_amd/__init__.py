"""MI355X-native (gfx950) VMonarch attention hot path.

Public API identical to the reference package `video_monarch_attention` (its __init__.py:1-4):
VMonarchAttention, vmonarch_attention, flash_entropy_attention.  Beside it, for models that attend causally and answer
token by token: packed_attention (whole prompts, forward and backward), and a paged key / value cache with the attention
of new tokens over it (paged_attention, append_pages, copy_pages, PagedKVCache).
"""
from .kernel import flash_entropy_attention
from .packed import packed_attention
from .paged import PagedKVCache, append_pages, copy_pages, paged_attention
from .vmonarch import VMonarchAttention, vmonarch_attention

__all__ = ["VMonarchAttention", "vmonarch_attention", "flash_entropy_attention", "packed_attention", "paged_attention",
           "append_pages", "copy_pages", "PagedKVCache"]
