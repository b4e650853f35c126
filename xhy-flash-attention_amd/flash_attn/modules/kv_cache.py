"""The key/value cache of one attention layer, as ``MHA.forward(..., kv_cache=cache)`` uses it.

    cache = KVCache(batch, slots, nheads_k, headdim, device="cuda", dtype=torch.bfloat16, track_weight=True)
    y = mha(x, kv_cache=cache)                        # x: the prompt, or the next tokens
    cache.accept(x.shape[1])
    y = mha(drafts, kv_cache=cache, tree_mask=mask, depth=mask.sum(-1, dtype=torch.int32) - 1)
    cache.commit(accepted)                            # of a tree of drafted tokens
    cache.evict(budget, sink=4, recent=256)

Lengths and positions live on the GPU and are updated in place: nothing here synchronises (but a rotary table
that grows), and a step captured into a graph goes on where its last replay stopped.
"""
import torch

from flash_attn.kvcache_interface import flash_attn_kvcache_commit_, flash_attn_kvcache_evict_

__all__ = ["KVCache"]


class KVCache:
    """k, v: (batch, slots, nheads_k, headdim), or pages with ``block_table`` (flash_attn_kvcache_func).

    seqlens: int32 (batch,), the keys held; positions: int32 (batch,), the position of the next token, which
    eviction leaves alone; most: no position is above it (known on the host: it sizes the rotary table.
    Replays of a graph do not count it up: set it to the longest length that they reach before the
    capture, as a position outside the table gives NaN); max_position: the longest that a sequence gets,
    which ``most`` stops at (a commit counts every drafted token into it, as the host does not know how
    many stay); attn_weight: fp32 (batch, nheads_k, slots) with track_weight, else None."""

    def __init__(self, batch_size, slots, nheads_k, headdim, device=None, dtype=None, track_weight=False,
                 max_position=None):
        self.k = torch.zeros(batch_size, slots, nheads_k, headdim, device=device, dtype=dtype)
        self.v = torch.zeros_like(self.k)
        self.block_table = None
        self.seqlens = torch.zeros(batch_size, device=device, dtype=torch.int32)
        self.positions = torch.zeros_like(self.seqlens)
        self.most, self.max_position = 0, max_position
        self._slot = torch.arange(slots, device=device, dtype=torch.int32)
        self.attn_weight = None
        if track_weight:
            self.attn_weight = torch.zeros(batch_size, nheads_k, slots, device=device, dtype=torch.float32)

    def clear_drafts(self):
        """Before a call: the weights of the slots behind the keys held become 0.  A call whose tokens were not
        kept has left theirs there, and the next call adds to them (what its tokens gave to the keys
        held stays: those were looked at)."""
        if self.attn_weight is None:
            return
        slot, columns = self._slot, self.attn_weight.shape[2]
        if slot.numel() != columns:                # weights of the caller's own
            slot = torch.arange(columns, device=slot.device, dtype=torch.int32)
        self.attn_weight.masked_fill_((slot >= self.seqlens[:, None])[:, None], 0.0)

    def _advance(self, count):
        self.most += count
        if self.max_position is not None:
            self.most = min(self.most, self.max_position)

    def _room(self):
        slots = self.k.shape[1] * (1 if self.block_table is None else self.block_table.shape[1])
        return slots if self.attn_weight is None else min(slots, self.attn_weight.shape[2])

    def accept(self, count):
        """Keeps all ``count`` tokens of the last call; a sequence that had no room for them stays as it is."""
        kept = self.seqlens <= self._room() - count
        self.seqlens.add_(kept, alpha=count)
        self.positions.add_(kept, alpha=count)
        self._advance(count)

    def commit(self, accepted):
        """Keeps the accepted ones (bool (batch, seqlen_q)) of the last call's tokens, in their order."""
        seqlens = flash_attn_kvcache_commit_(self.k, self.v, self.seqlens, accepted, self.block_table, self.attn_weight)
        self.positions += seqlens - self.seqlens
        self.seqlens.copy_(seqlens)
        self._advance(accepted.shape[1])

    def evict(self, budget, sink=0, recent=0):
        """Shrinks sequences of more than ``budget`` keys; returns the slots the kept keys came from."""
        if self.attn_weight is None:
            raise RuntimeError("KVCache: eviction needs track_weight=True")
        seqlens, weight, kept = flash_attn_kvcache_evict_(self.k, self.v, self.seqlens, self.attn_weight, budget, sink,
                                                          recent, self.block_table)
        self.seqlens.copy_(seqlens)
        self.attn_weight.copy_(weight)
        return kept
