"""Key/value cache for serving: attention of drafted tokens over it, commit, eviction.

    out = flash_attn_kvcache_func(q, k_cache, v_cache, cache_seqlens, k=k, v=v, tree_mask=mask)
    cache_seqlens = flash_attn_kvcache_commit_(k_cache, v_cache, cache_seqlens, accepted)
    cache_seqlens, attn_weight, kept = flash_attn_kvcache_evict_(k_cache, v_cache, cache_seqlens,
                                                                 attn_weight, budget)

The cache is (batch, slots, nheads_k, headdim) or, with a block table, pages of (num_pages, page_size,
nheads_k, headdim).  Lengths and block table stay on the device: no call synchronises, every call can be
captured in a graph, and no kernel touches memory outside the cache whatever they hold.  A tensor that a
call writes may not be expanded or share memory with another that it writes.  The checks and allocations
are in C++ (csrc/fa_host.cpp: a decoding step is short); the kernels are behind ``flash_attn_kvcache``,
``flash_attn_kvcache_commit`` and ``flash_attn_kvcache_evict`` (include/flash_attn.h); no reference
counterpart (the reference's 2.0.8 API has no cache).
"""
import flash_attn_2_cuda as _ext

__all__ = ["flash_attn_kvcache_func", "flash_attn_kvcache_commit_", "flash_attn_kvcache_evict_"]


def flash_attn_kvcache_func(q, k_cache, v_cache, cache_seqlens, k=None, v=None, block_table=None, tree_mask=None,
                            softmax_scale=None, attn_weight=None, return_softmax_lse=False):
    """Attention of seqlen_q drafted tokens (1: plain decoding) over a key/value cache.

    The drafted tokens of sequence i follow its cache_seqlens[i] cached keys: each sees all of those,
    and of the drafted tokens the ones that tree_mask names (default: itself and those before it).

    Arguments:
        q: (batch, seqlen_q, nheads, headdim), fp16 or bf16; nheads a multiple of nheads_k.
        k_cache, v_cache: (batch, slots, nheads_k, headdim), or pages (num_pages, page_size, nheads_k,
            headdim) with block_table int32 (batch, blocks); headdim a multiple of 8, at most 256;
            equal strides, 16-byte aligned.
        cache_seqlens: int32 (batch,), the keys in the cache before the drafted ones.
        k, v: (batch, seqlen_q, nheads_k, headdim), the drafted tokens' keys and values: stored into the
            slots behind the cached ones by the same call.  None: they are there already.
        tree_mask: bool (seqlen_q, seqlen_q) or (batch, seqlen_q, seqlen_q), row: who sees, column: who is
            seen.  A drafted token that no row sees may hold anything.
        softmax_scale: default 1 / sqrt(headdim).
        attn_weight: fp32 (batch, nheads_k, slots), optional: every key's entry grows by the sum of its
            probabilities over the rows of the query heads that share the kv head, the drafted tokens' entries
            among them: they should hold 0 before (commit and eviction leave it so; after a call whose tokens
            are not kept, KVCache.clear_drafts does).  With fewer columns than the cache has slots, sequences
            have room for as many keys (in the other calls too).
        return_softmax_lse: also return the log-sum-exp of the scaled scores, fp32 (batch, nheads, seqlen_q).
    cache_seqlens is not changed (flash_attn_kvcache_commit_ gives the new lengths).  A row that sees
    no key gives 0 and +inf.  A sequence whose length leaves no room for the drafted tokens, or that
    names a page outside the cache, gives NaN; of the former nothing is stored or added.  No backward."""
    out, lse = _ext.host_module().kvcache(q, k_cache, v_cache, cache_seqlens, k, v, block_table, tree_mask,
                                          softmax_scale, attn_weight)
    return (out, lse) if return_softmax_lse else out


def flash_attn_kvcache_commit_(k_cache, v_cache, cache_seqlens, accepted, block_table=None, attn_weight=None):
    """Keeps the accepted ones of the drafted tokens behind the cached keys, in place.

    accepted: bool (batch, seqlen_q), the drafted tokens that stay; their keys and values move to the
    slots right behind the cached keys, in their order.  attn_weight (as flash_attn_kvcache_func) moves
    along, and the drafted slots behind the kept ones become 0.  Returns the new lengths, int32 (batch,).
    A sequence whose length leaves no room for the drafted tokens stays as it is.  With a block table no
    page may belong to two sequences."""
    return _ext.host_module().commit(k_cache, v_cache, cache_seqlens, accepted, block_table, attn_weight)


def flash_attn_kvcache_evict_(k_cache, v_cache, cache_seqlens, attn_weight, budget, sink=0, recent=0,
                              block_table=None):
    """Shrinks every sequence of more than ``budget`` keys to ``budget``, in place.

    Each kv head keeps the first ``sink`` keys, the last ``recent``, and of the others those with the
    largest attn_weight (fp32 (batch, nheads_k, slots); equal weights: the lowest slot), sink + recent <=
    budget.  Kept keys move to slots 0 .. budget - 1 in their order (their rotary embedding stays that of
    the position they were written at).

    Returns (cache_seqlens, attn_weight, kept): the new lengths; the kept keys' weights in their new
    slots and 0 behind them, a new tensor; and kept, int32 (batch, nheads_k, budget), the slot each kept
    key came from (-1 behind the last).  A sequence whose length is not in [0, slots] stays as it is.
    With a block table no page may belong to two sequences."""
    return _ext.host_module().evict(k_cache, v_cache, cache_seqlens, attn_weight, budget, sink, recent,
                                    block_table)
