"""B200-native flash attention (forward + backward) with an optional trainable bias.

Public interface (same names and signatures as the reference project):
    flash_attention_fn, flash_attention_qkvpacked_fn,
    FlashAttentionFn, FlashAttentionQKVPackedFn
plus, with no counterpart in the reference: FlashAttention (nn.Module), flash_attention_op
(the same call through torch.library operators), shard_batch_heads, and for serving a paged key / value
cache: PagedKVCache, paged_attention_fn, paged_kv_extend, paged_kv_write, paged_kv_release (and
paged_attention_op, paged_kv_write_op through torch.library).
"""
from .flash_attention import (  # noqa: F401
    FlashAttentionFn,
    FlashAttentionQKVPackedFn,
    flash_attention_fn,
    flash_attention_qkvpacked_fn,
)
from .module import FlashAttention, flash_attention_op, paged_attention_op, paged_kv_write_op  # noqa: F401
from .paged import (  # noqa: F401
    PagedKVCache,
    paged_attention_fn,
    paged_kv_extend,
    paged_kv_release,
    paged_kv_write,
)
from .sharding import shard_batch_heads  # noqa: F401

__all__ = [
    "FlashAttentionFn",
    "FlashAttentionQKVPackedFn",
    "flash_attention_fn",
    "flash_attention_qkvpacked_fn",
    "FlashAttention",
    "flash_attention_op",
    "shard_batch_heads",
    "PagedKVCache",
    "paged_attention_fn",
    "paged_attention_op",
    "paged_kv_extend",
    "paged_kv_release",
    "paged_kv_write",
    "paged_kv_write_op",
]
