"""Key/value cache for serving: attention of drafted tokens over it, commit, eviction.

    out = flash_attn_kvcache_func(q, k_cache, v_cache, cache_seqlens, k=k, v=v, tree_mask=mask)
    cache_seqlens = flash_attn_kvcache_commit_(k_cache, v_cache, cache_seqlens, accepted)
    cache_seqlens, attn_weight, kept = flash_attn_kvcache_evict_(k_cache, v_cache, cache_seqlens,
                                                                 attn_weight, budget)

The cache is (batch, slots, nheads_k, headdim) or, with a block table, pages of (num_pages, page_size,
nheads_k, headdim).  Lengths and block table stay on the device: no call synchronises, every call can be
captured in a graph, and no kernel touches memory outside the cache whatever they hold.  The kernels
are behind ``flash_attn_kvcache``, ``flash_attn_kvcache_commit`` and ``flash_attn_kvcache_evict``
(include/flash_attn.h); no reference counterpart (the reference's 2.0.8 API has no cache).
"""
from __future__ import annotations

import ctypes

import torch

import flash_attn_2_cuda as _ext

__all__ = ["flash_attn_kvcache_func", "flash_attn_kvcache_commit_", "flash_attn_kvcache_evict_"]

_lib = _ext._lib
_P, _I, _I64, _F, _B = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_bool
_lib.flash_attn_kvcache.argtypes = [_P] * 12 + [_I] * 8 + [_F] + [_P] * 5 + [_I64] + [_P] * 2 + [_B, _P]
_lib.flash_attn_kvcache.restype = _B
_lib.flash_attn_kvcache_workspace.argtypes = [_I] * 6 + [_B]
_lib.flash_attn_kvcache_workspace.restype = ctypes.c_size_t
_lib.flash_attn_kvcache_evict.argtypes = [_P] * 9 + [_I] * 9 + [_P, _I64, _P, _P, _P]
_lib.flash_attn_kvcache_evict.restype = _B
_lib.flash_attn_kvcache_commit.argtypes = [_P] * 7 + [_I] * 7 + [_P, _I64, _I64, _P, _P]
_lib.flash_attn_kvcache_commit.restype = _B


def _ints(*x):
    return (_I64 * len(x))(*x)


def _cache_args(k_cache, v_cache, cache_seqlens, block_table):
    """Checks the cache; returns (batch, slots, page_size, num_pages, strides, table stride)."""
    check = _ext._check
    check(k_cache.dtype in (torch.float16, torch.bfloat16), "kvcache: only fp16 and bf16 are supported")
    check(v_cache.dtype == k_cache.dtype, "kvcache: k_cache and v_cache must have the same dtype")
    check(k_cache.dim() == 4 and v_cache.shape == k_cache.shape,
          "kvcache: k_cache and v_cache must both be (batch or pages, slots, nheads_k, headdim)")
    check(k_cache.numel() > 0, "kvcache: the cache is empty")
    check(v_cache.stride() == k_cache.stride(), "kvcache: k_cache and v_cache must have the same strides")
    d = k_cache.shape[3]
    check(d % 8 == 0 and d <= 256, "kvcache: headdim must be a multiple of 8, at most 256")
    check(k_cache.stride(3) == 1, "kvcache: the cache must have a contiguous last dimension")
    check(_ext._aligned(k_cache) and _ext._aligned(v_cache),
          "kvcache: the cache must be 16-byte aligned in its base and strides")
    check(cache_seqlens.dtype == torch.int32 and cache_seqlens.dim() == 1 and cache_seqlens.is_contiguous(),
          "kvcache: cache_seqlens must be a contiguous int32 vector")
    b = cache_seqlens.shape[0]
    check(b > 0, "kvcache: batch size must be positive")
    strides = _ints(*k_cache.stride()[:3])
    if block_table is None:
        check(k_cache.shape[0] == b, "kvcache: the cache and cache_seqlens must have the same batch size")
        return b, k_cache.shape[1], 0, 0, strides, 0
    check(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == b,
          "kvcache: block_table must be int32 (batch, blocks)")
    check(block_table.shape[1] > 0 and block_table.stride(1) == 1,
          "kvcache: block_table must have a contiguous last dimension")
    slots = block_table.shape[1] * k_cache.shape[1]
    check(slots < 2 ** 31 - 256, "kvcache: too many slots")
    return b, slots, k_cache.shape[1], k_cache.shape[0], strides, block_table.stride(0)


def _check_device(*tensors):
    """Last of the checks: everything on one gfx950 GPU."""
    tensors = [t for t in tensors if t is not None]
    _ext._check(all(t.is_cuda for t in tensors), "kvcache: tensors must be on the GPU")
    _ext._check(all(t.device == tensors[0].device for t in tensors), "kvcache: tensors must share a device")
    _ext._check(_ext._is_gfx950(tensors[0].device), "kvcache: only gfx950 (MI355X) GPUs are supported")


def _check_weight(w, b, hk, slots):
    """Returns the slots that a call with these weights has room for."""
    _ext._check(w.dtype == torch.float32 and w.dim() == 3 and tuple(w.shape[:2]) == (b, hk) and w.shape[2] > 0,
                "kvcache: attn_weight must be fp32 (batch, nheads_k, slots)")
    _ext._check(w.stride(2) == 1, "kvcache: attn_weight must have a contiguous last dimension")
    return min(slots, w.shape[2])


def _flag_bytes(m, shape, name):
    _ext._check(m.dtype == torch.bool and tuple(m.shape) in shape, f"kvcache: {name} must be bool {shape[-1]}")
    return m if m.stride(-1) == 1 else m.contiguous()


def _check_no_grad(*tensors):
    _ext._check(not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)),
                "kvcache: the cache has no backward; call it under torch.no_grad()")


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
            probabilities over the rows of the query heads that share the kv head.  With fewer columns
            than the cache has slots, sequences have room for as many keys (in the other calls too).
        return_softmax_lse: also return the log-sum-exp of the scaled scores, fp32 (batch, nheads, seqlen_q).
    cache_seqlens is not changed (flash_attn_kvcache_commit_ gives the new lengths).  A row that sees
    no key gives 0 and +inf.  A sequence whose length leaves no room for the drafted tokens, or that
    names a page outside the cache, gives NaN; of the former nothing is stored or added.  No backward."""
    check = _ext._check
    b, slots, page, pages, cstr, tstr = _cache_args(k_cache, v_cache, cache_seqlens, block_table)
    check(q.dtype == k_cache.dtype, "kvcache: q and the cache must have the same dtype")
    hk, d = k_cache.shape[2:]
    check(q.dim() == 4 and q.shape[0] == b and q.shape[3] == d,
          "kvcache: q must have shape (batch, seqlen_q, nheads, headdim)")
    sq, h = q.shape[1:3]
    if attn_weight is not None:
        slots = _check_weight(attn_weight, b, hk, slots)
    check(sq > 0, "kvcache: at least one drafted token")
    check(h > 0 and h % hk == 0, "Number of heads in key/value must divide number of heads in query")
    check(sq <= slots, "kvcache: more drafted tokens than slots")
    check((k is None) == (v is None), "kvcache: k and v come together")
    check(q.stride(3) == 1, "kvcache: q must have a contiguous last dimension")
    if k is not None:
        for t in (k, v):
            check(t.dtype == q.dtype, "kvcache: k and v must have the cache's dtype")
            check(tuple(t.shape) == (b, sq, hk, d), "kvcache: k and v must have shape (batch, seqlen_q, nheads_k, headdim)")
            check(t.stride(3) == 1, "kvcache: k and v must have a contiguous last dimension")
    _check_no_grad(q, k, v, k_cache, v_cache)
    if tree_mask is not None:
        tree_mask = _flag_bytes(tree_mask, ((sq, sq), (b, sq, sq)), "tree_mask")
        mstr = _ints(tree_mask.stride(0) if tree_mask.dim() == 3 else 0, tree_mask.stride(-2))
    scale = d ** -0.5 if softmax_scale is None else float(softmax_scale)
    check(0.0 < scale < float("inf"), "kvcache: softmax_scale must be positive and finite")
    _check_device(k_cache, v_cache, cache_seqlens, block_table, q, k, v, tree_mask, attn_weight)
    q = _ext._vec_ok(q)
    if k is not None:
        k, v = _ext._vec_ok(k), _ext._vec_ok(v)
    ptr = _ext._ptr
    with _ext._device_guard(q.device):
        out = torch.empty((b, sq, h, d), dtype=q.dtype, device=q.device)
        lse = torch.empty((b, h, sq), dtype=torch.float32, device=q.device)
        size = _lib.flash_attn_kvcache_workspace(b, sq, slots, h, hk, d, attn_weight is not None)
        work = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        none = _ints(0, 0, 0)
        ok = _lib.flash_attn_kvcache(
            ptr(q), ptr(k_cache), ptr(v_cache), ptr(k), ptr(v), ptr(out), ptr(lse), ptr(attn_weight),
            ptr(cache_seqlens), ptr(block_table), ptr(tree_mask), ptr(work), b, sq, slots, h, hk, d, page, pages, scale,
            _ints(*q.stride()[:3]), cstr, none if k is None else _ints(*k.stride()[:3]),
            none if v is None else _ints(*v.stride()[:3]), _ints(*out.stride()[:3]), tstr,
            none if tree_mask is None else mstr, none if attn_weight is None else _ints(*attn_weight.stride()[:2]),
            q.dtype == torch.bfloat16, _ext._stream(q))
        if not ok:
            _ext._raise_lib_error("flash_attn_kvcache")
    return (out, lse) if return_softmax_lse else out


def flash_attn_kvcache_commit_(k_cache, v_cache, cache_seqlens, accepted, block_table=None, attn_weight=None):
    """Keeps the accepted ones of the drafted tokens behind the cached keys, in place.

    accepted: bool (batch, seqlen_q), the drafted tokens that stay; their keys and values move to the
    slots right behind the cached keys, in their order.  attn_weight (as flash_attn_kvcache_func) moves
    along, and the drafted slots behind the kept ones become 0.  Returns the new lengths, int32 (batch,).
    A sequence whose length leaves no room for the drafted tokens stays as it is.  With a block table no
    page may belong to two sequences."""
    b, slots, page, pages, cstr, tstr = _cache_args(k_cache, v_cache, cache_seqlens, block_table)
    hk, d = k_cache.shape[2:]
    _ext._check(accepted.dim() == 2 and accepted.shape[0] == b, "kvcache: accepted must be bool (batch, seqlen_q)")
    sq = accepted.shape[1]
    if attn_weight is not None:
        slots = _check_weight(attn_weight, b, hk, slots)
    _ext._check(0 < sq <= 8192 and sq <= slots, "kvcache: between 1 and min(8192, slots) drafted tokens")
    accepted = _flag_bytes(accepted, ((b, sq),), "accepted")
    _check_no_grad(k_cache, v_cache)
    _check_device(k_cache, v_cache, cache_seqlens, block_table, accepted, attn_weight)
    ptr = _ext._ptr
    with _ext._device_guard(k_cache.device):
        lens = torch.empty_like(cache_seqlens)
        ok = _lib.flash_attn_kvcache_commit(
            ptr(k_cache), ptr(v_cache), ptr(cache_seqlens), ptr(accepted), ptr(block_table), ptr(lens), ptr(attn_weight),
            b, sq, slots, hk, d, page, pages, cstr, tstr, accepted.stride(0),
            _ints(0, 0) if attn_weight is None else _ints(*attn_weight.stride()[:2]), _ext._stream(k_cache))
        if not ok:
            _ext._raise_lib_error("flash_attn_kvcache_commit")
    return lens


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
    b, slots, page, pages, cstr, tstr = _cache_args(k_cache, v_cache, cache_seqlens, block_table)
    hk, d = k_cache.shape[2:]
    budget, sink, recent = int(budget), int(sink), int(recent)
    _ext._check(0 < budget < 2 ** 31 and sink >= 0 and recent >= 0 and sink + recent <= budget,
                "kvcache: budget must be positive and at least sink + recent")
    _ext._check(b <= 65535, "kvcache: batch size must be at most 65535")
    slots = _check_weight(attn_weight, b, hk, slots)
    _check_no_grad(k_cache, v_cache, attn_weight)
    _check_device(k_cache, v_cache, cache_seqlens, block_table, attn_weight)
    ptr = _ext._ptr
    dev = k_cache.device
    with _ext._device_guard(dev):
        lens = torch.empty_like(cache_seqlens)
        weight = torch.empty((b, hk, attn_weight.shape[2]), dtype=torch.float32, device=dev)
        if attn_weight.shape[2] > slots:
            weight[:, :, slots:] = attn_weight[:, :, slots:]
        kept = torch.empty((b, hk, budget), dtype=torch.int32, device=dev)
        work = torch.empty(b * hk, dtype=torch.int32, device=dev)
        ok = _lib.flash_attn_kvcache_evict(
            ptr(k_cache), ptr(v_cache), ptr(cache_seqlens), ptr(attn_weight), ptr(block_table), ptr(lens), ptr(weight),
            ptr(kept), ptr(work), b, slots, hk, d, page, pages, budget, sink, recent, cstr, tstr,
            _ints(*attn_weight.stride()[:2]), _ints(*weight.stride()[:2]), _ext._stream(k_cache))
        if not ok:
            _ext._raise_lib_error("flash_attn_kvcache_evict")
    return lens, weight, kept
