"""A paged key / value cache and the attention of new tokens over it, for serving.

The cache is `pages` pages of `page_size` tokens; a sequence holds pages anywhere in it, named by its row of a block table, so
sequences grow and end without copies.  All of it runs on the GPU, on the current stream and without synchronisation: lengths,
tables and the stack of free pages are device tensors, so a whole decode step can be captured into a CUDA graph.

    paged_kv_extend     pages and slots for each request's new tokens, from the request lengths
    paged_kv_write      the new tokens' keys and values into their slots
    paged_attention_fn  attention of one new token a sequence over its pages
    paged_kv_release    the pages of finished requests back on the stack
    PagedKVCache        the tensors that these work on, with the four as methods

None of them has a derivative: an input that requires grad is refused outside torch.no_grad().  The reference project has no
counterpart.  The compute path is libfa_sm100.so, as for `flash_attention_fn`.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .flash_attention import _native


def paged_attention_fn(q, k_cache, v_cache, block_table, seq_lens, bias=None, sm_scale=None) -> torch.Tensor:
    """Attention of one new token a sequence; returns (B, H, D) in q's dtype.

    q                 (B, H, D) fp16 / bf16, D one of 16, 32, 64, 128, 256
    k_cache, v_cache  (pages, page_size, Hkv, D) in q's dtype, H a multiple of Hkv: head h reads key head h // (H // Hkv).  Any
                      strides that are multiples of 16 bytes (a (pages, Hkv, page_size, D) cache transposed, a layer's slice)
    block_table       (B, W) int32: the key at position n lies in row n % page_size of page block_table[b, n // page_size]
    seq_lens          (B,) int32: keys of each sequence, the new token's own among them (write it first)
    bias              (B, H, W * page_size), as in `flash_attention_fn`: bool (False is left out) or float (added to the scaled
                      scores); expanded views are read in place, other float dtypes than q's as fp32 (converted, fp32 itself
                      apart, and so are other inner strides copied: what there is of an expanded view)
    sm_scale          None: 1 / sqrt(D)

    A sequence of length 0 and a row whose mask leaves nothing give 0.  What a mask or a bias of -inf leaves out takes no part,
    whatever its key and value hold; so do keys on a page that the cache does not have, and lengths are cut to what the table
    has room for.  The keys are split over the GPU by the lengths of the call: the same call gives the same bits, but a
    sequence's last bits may change with the others beside it.
    """
    return _native.paged_attention(q, k_cache, v_cache, block_table, seq_lens, bias, sm_scale)


def paged_kv_write(k, v, k_cache, v_cache, slot_mapping) -> None:
    """Writes k, v (T, Hkv, D) into the caches (pages, page_size, Hkv, D), token t into row slot % page_size of page
    slot // page_size with slot = slot_mapping[t] (int64).  Tokens with a slot below 0 or behind the cache are not written.  The
    slots of a call must differ from one another: of two tokens with one slot, parts of both may stay.  Rows of the cache itself
    can be given (a page copied to another, tokens moved): they are copied first, so each slot gets what was there before the
    call."""
    _native.paged_kv_write(k, v, k_cache, v_cache, slot_mapping)


def paged_kv_extend(block_table, seq_lens, new_lens, free_pages, free_count, page_size: int, num_tokens: int,
                    inplace: bool = False) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Room for new tokens; returns (slot_mapping (num_tokens,) int64, seq_lens after, free_count after).

    block_table  (B, W) int32; gets the new pages, in place
    seq_lens     (B,) int32: tokens held; new_lens (B,) int32: tokens that come (below 0 counts as 0)
    free_pages   (F,) int32: a stack, of which free_pages[:free_count] are free; free_count one int32.  Taken from the top
    num_tokens   rows of the call: the new tokens of all requests lie one request after the other, the rest is padding (slot -1)
    inplace      write the lengths and the count into seq_lens and free_count themselves

    Requests are served in order.  One whose tokens do not fit its row of the table, or reach beyond num_tokens, gets nothing:
    its length stays and its tokens' slots are -1.  From the first request on that finds too few free pages, those that need
    pages get nothing either.
    """
    return _native.paged_kv_extend(block_table, seq_lens, new_lens, free_pages, free_count, page_size, num_tokens, inplace)


def paged_kv_release(block_table, seq_lens, finished, free_pages, free_count, page_size: int,
                     inplace: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Puts the pages of the requests with finished[b] (bool) back on the stack, in order, in place in free_pages; returns
    (seq_lens after, 0 for the finished; free_count after).  The table is only read.

    Lengths and table of a finished request must be what `paged_kv_extend` made them, and no two finished requests may hold the
    same page: what goes back is not looked at, and a page that is on the stack twice, or was never taken from it, is given to two
    requests later on."""
    return _native.paged_kv_release(block_table, seq_lens, finished, free_pages, free_count, page_size, inplace)


class PagedKVCache:
    """The caches of a model's layers with one block table for all of them.

        cache = PagedKVCache(layers, pages, page_size, Hkv, D, max_seqs, max_len)
        slots = cache.extend(new_lens, num_tokens)         # once a step
        cache.write(layer, k, v, slots)                    # k, v (num_tokens, Hkv, D)
        out = cache.attend(layer, q)                       # q (max_seqs, H, D): one new token a sequence
        cache.release(finished)                            # (max_seqs,) bool

    k, v          (layers, pages, page_size, Hkv, D)
    block_table   (max_seqs, ceil(max_len / page_size)) int32, seq_lens (max_seqs,) int32
    free_pages    (pages,) int32, free_count (1,) int32
    All tensors stay at their addresses and are updated in place.
    """

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, max_seqs: int,
                 max_len: int, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        for name, x in (("num_layers", num_layers), ("num_pages", num_pages), ("page_size", page_size),
                        ("num_kv_heads", num_kv_heads), ("max_seqs", max_seqs), ("max_len", max_len)):
            if x < 1:
                raise ValueError(f"{name} must be at least 1, got {x}")
        if head_dim not in (16, 32, 64, 128, 256):
            raise AssertionError("head dimension must be one of 16, 32, 64, 128, 256")
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError("the cache's dtype must be torch.float16 or torch.bfloat16")
        self.page_size = page_size
        shape = (num_layers, num_pages, page_size, num_kv_heads, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        ints = dict(dtype=torch.int32, device=device)
        self.block_table = torch.zeros((max_seqs, -(-max_len // page_size)), **ints)
        self.seq_lens = torch.zeros((max_seqs,), **ints)
        self.free_pages = torch.arange(num_pages, **ints)
        self.free_count = torch.full((1,), num_pages, **ints)

    def extend(self, new_lens: torch.Tensor, num_tokens: int) -> torch.Tensor:
        """Slots for new_lens[b] more tokens of each sequence (see `paged_kv_extend`)."""
        return paged_kv_extend(self.block_table, self.seq_lens, new_lens, self.free_pages, self.free_count, self.page_size,
                               num_tokens, inplace=True)[0]

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor) -> None:
        paged_kv_write(k, v, self.k[layer], self.v[layer], slot_mapping)

    def attend(self, layer: int, q: torch.Tensor, bias: Optional[torch.Tensor] = None,
               sm_scale: Optional[float] = None) -> torch.Tensor:
        return paged_attention_fn(q, self.k[layer], self.v[layer], self.block_table, self.seq_lens, bias, sm_scale)

    def release(self, finished: torch.Tensor) -> None:
        paged_kv_release(self.block_table, self.seq_lens, finished, self.free_pages, self.free_count, self.page_size, inplace=True)
