"""Attention modules over the MI355X kernels (the reference's callers).

Drop-in for the attention-core classes of the reference's ``flash_attn/modules/mha.py``:

  * ``FlashSelfAttention``  (reference ``:35-84``)   -- packed qkv, fixed-length or varlen;
  * ``FlashCrossAttention`` (reference ``:87-142``)  -- q plus packed kv, fixed-length or varlen;
  * ``MHA``                 (reference ``:343-561``) -- the projection wrapper, restricted to what
    sits on this path: fused Wqkv (or Wq + Wkv for cross attention), MQA / GQA through
    ``num_heads_kv``, rotary embedding (``flash_attn.layers.rotary``, HIP kernel), causal /
    dropout / softmax_scale, and the output projection; beyond the reference, ``qk_norm`` (per-head
    RMS norm of q and k in the rotary's pass, ``flash_attn.layers.qk_norm``) and generation over a
    ``flash_attn.modules.kv_cache.KVCache``.  The reference's tensor-parallel linears, fused dense and
    ``inference_params`` are out of scope (SURVEY.md §8 marks the callers' own
    subsystems outside the hot path); asking for them raises.

Same constructor arguments, forward signatures, shape conventions and dropout semantics
(``self.drop.p`` while training, 0 in eval) as the reference.  Everything runs through
``flash_attn.flash_attn_interface`` -- there is no PyTorch fallback attention here.
"""
import torch
import torch.nn as nn

from flash_attn.flash_attn_interface import (flash_attn_func, flash_attn_kvpacked_func, flash_attn_qkvpacked_func,
                                             flash_attn_varlen_func, flash_attn_varlen_kvpacked_func,
                                             flash_attn_varlen_qkvpacked_func)
from flash_attn.kvcache_interface import flash_attn_kvcache_func

__all__ = ["FlashSelfAttention", "FlashCrossAttention", "MHA"]


class FlashSelfAttention(nn.Module):
    """Scaled dot-product attention with softmax over packed qkv (reference mha.py:35-84).

    softmax_scale: temperature (default 1/sqrt(headdim)); attention_dropout: dropout rate.
    """

    def __init__(self, causal=False, softmax_scale=None, attention_dropout=0.0):
        super().__init__()
        self.causal = causal
        self.softmax_scale = softmax_scale
        self.drop = nn.Dropout(attention_dropout)

    def forward(self, qkv, causal=None, cu_seqlens=None, max_seqlen=None):
        """qkv: (B, S, 3, H, D), or (total, 3, H, D) with cu_seqlens (B+1,) int32 and max_seqlen.
        Returns (B, S, H, D), or (total, H, D) for varlen."""
        assert qkv.dtype in (torch.float16, torch.bfloat16)
        assert qkv.is_cuda
        causal = self.causal if causal is None else causal
        dropout_p = self.drop.p if self.training else 0.0
        if cu_seqlens is not None:
            assert cu_seqlens.dtype == torch.int32
            assert max_seqlen is not None and isinstance(max_seqlen, int)
            return flash_attn_varlen_qkvpacked_func(qkv, cu_seqlens, max_seqlen, dropout_p,
                                                    softmax_scale=self.softmax_scale, causal=causal)
        return flash_attn_qkvpacked_func(qkv, dropout_p, softmax_scale=self.softmax_scale, causal=causal)


class FlashCrossAttention(nn.Module):
    """Scaled dot-product attention of q against packed kv (reference mha.py:87-142)."""

    def __init__(self, causal=False, softmax_scale=None, attention_dropout=0.0):
        super().__init__()
        self.causal = causal
        self.softmax_scale = softmax_scale
        self.drop = nn.Dropout(attention_dropout)

    def forward(self, q, kv, causal=None, cu_seqlens=None, max_seqlen=None, cu_seqlens_k=None,
                max_seqlen_k=None):
        """q: (B, Sq, H, D), kv: (B, Sk, 2, H_k, D); varlen: q (total_q, H, D), kv (total_k, 2, H_k, D)
        with cu_seqlens / cu_seqlens_k (B+1,) int32 and max_seqlen / max_seqlen_k."""
        assert q.dtype in (torch.float16, torch.bfloat16)
        assert q.is_cuda and kv.is_cuda
        causal = self.causal if causal is None else causal
        dropout_p = self.drop.p if self.training else 0.0
        if cu_seqlens is not None:
            assert cu_seqlens.dtype == torch.int32
            assert max_seqlen is not None and isinstance(max_seqlen, int)
            assert cu_seqlens_k is not None and cu_seqlens_k.dtype == torch.int32
            assert max_seqlen_k is not None and isinstance(max_seqlen_k, int)
            return flash_attn_varlen_kvpacked_func(q, kv, cu_seqlens, cu_seqlens_k, max_seqlen,
                                                   max_seqlen_k, dropout_p,
                                                   softmax_scale=self.softmax_scale, causal=causal)
        batch_size = q.shape[0]
        assert kv.shape[0] == batch_size and kv.shape[4] == q.shape[3]
        return flash_attn_kvpacked_func(q, kv, dropout_p, softmax_scale=self.softmax_scale,
                                        causal=causal)


class MHA(nn.Module):
    """Multi-head attention block: Wqkv -> FlashSelfAttention / FlashCrossAttention -> out_proj.

    Constructor arguments follow the reference (mha.py:347-448, forward :449-561); rotary_emb_dim > 0
    applies flash_attn.layers.rotary.RotaryEmbedding (HIP kernel) to q and k as the reference does.
    qk_norm puts an RMS norm with a learned weight on each head of q and k, before the rotary embedding.
    The ones that select subsystems outside this build (fused_bias_fc, dwconv, return_residual,
    process_group, use_flash_attn=False) are accepted only at their neutral value.
    """

    def __init__(self, embed_dim, num_heads, num_heads_kv=None, cross_attn=False, qkv_proj_bias=True,
                 out_proj_bias=True, dropout=0.0, softmax_scale=None, causal=False, layer_idx=None,
                 dwconv=False, rotary_emb_dim=0, rotary_emb_base=10000.0, rotary_emb_scale_base=None,
                 rotary_emb_interleaved=False, fused_bias_fc=False, use_flash_attn=True,
                 return_residual=False, checkpointing=False, device=None, dtype=None, qk_norm=False,
                 qk_norm_eps=1e-6):
        super().__init__()
        for name, val, neutral in (("dwconv", dwconv, False),
                                   ("fused_bias_fc", fused_bias_fc, False),
                                   ("use_flash_attn", use_flash_attn, True),
                                   ("return_residual", return_residual, False)):
            if val != neutral:
                raise NotImplementedError(f"MHA({name}={val!r}) is outside the MI355X attention build")
        factory = {"device": device, "dtype": dtype}
        self.embed_dim = embed_dim
        self.cross_attn = cross_attn
        self.causal = causal
        self.layer_idx = layer_idx
        self.checkpointing = checkpointing
        self.num_heads = num_heads
        self.num_heads_kv = num_heads_kv if num_heads_kv is not None else num_heads
        assert self.num_heads % self.num_heads_kv == 0, "num_heads must be divisible by num_heads_kv"
        assert self.embed_dim % num_heads == 0, "embed_dim must be divisible by num_heads"
        self.head_dim = self.embed_dim // num_heads
        self.rotary_emb_dim = rotary_emb_dim
        self.qk_norm = None
        if qk_norm:
            if cross_attn or rotary_emb_scale_base is not None:
                raise NotImplementedError("MHA(qk_norm=True) with cross attention or XPos scaling")
            from flash_attn.layers.qk_norm import QKNormRotary
            self.qk_norm = QKNormRotary(self.head_dim, rotary_emb_dim, base=rotary_emb_base,
                                        interleaved=rotary_emb_interleaved, eps=qk_norm_eps, device=device,
                                        dtype=dtype)
        elif rotary_emb_dim > 0:   # reference mha.py:379-384
            assert not cross_attn, "MHA with rotary embedding does not support cross-attention yet"
            from flash_attn.layers.rotary import RotaryEmbedding
            self.rotary_emb = RotaryEmbedding(rotary_emb_dim, base=rotary_emb_base,
                                              scale_base=rotary_emb_scale_base,
                                              interleaved=rotary_emb_interleaved, device=device)
        qkv_dim = self.head_dim * (self.num_heads + 2 * self.num_heads_kv)
        kv_dim = 2 * self.head_dim * self.num_heads_kv
        if not self.cross_attn:
            self.Wqkv = nn.Linear(embed_dim, qkv_dim, bias=qkv_proj_bias, **factory)
        else:
            self.Wq = nn.Linear(embed_dim, embed_dim, bias=qkv_proj_bias, **factory)
            self.Wkv = nn.Linear(embed_dim, kv_dim, bias=qkv_proj_bias, **factory)
        self.inner_attn = FlashSelfAttention(causal=causal, softmax_scale=softmax_scale,
                                             attention_dropout=dropout)
        self.inner_cross_attn = FlashCrossAttention(causal=causal, softmax_scale=softmax_scale,
                                                    attention_dropout=dropout)
        self.out_proj = nn.Linear(embed_dim, embed_dim, bias=out_proj_bias, **factory)

    def forward(self, x, x_kv=None, key_padding_mask=None, cu_seqlens=None, max_seqlen=None,
                mixer_subset=None, inference_params=None, kv_cache=None, tree_mask=None, depth=None, **kwargs):
        """x: (B, S, E), or (total, E) with cu_seqlens / max_seqlen (varlen, self-attention only).
        x_kv: (B, Sk, E) for cross attention.  key_padding_mask is the reference's padded-batch
        convenience: it unpads, runs varlen attention and pads back.
        kv_cache: a KVCache; x are the tokens behind its keys, which are stored (kv_cache.accept or .commit
        keeps them), and each attends to the cached keys and to those before it, or to what tree_mask
        names (flash_attn_kvcache_func).  depth: int32 (B, S), the tokens' distance from the first one's
        position (default 0 .. S - 1).  Causal self-attention only, under torch.no_grad()."""
        if kv_cache is not None:
            assert x_kv is None and key_padding_mask is None and cu_seqlens is None
            return self._forward_cached(x, kv_cache, tree_mask, depth)
        assert tree_mask is None and depth is None, "tree_mask and depth belong to a call with kv_cache"
        if inference_params is not None or mixer_subset is not None:
            raise NotImplementedError("MHA inference cache / mixer_subset is outside the MI355X build")
        if key_padding_mask is not None:
            assert cu_seqlens is None and not self.cross_attn
            from flash_attn.bert_padding import pad_input, unpad_input
            b, s = x.shape[:2]
            x_unpad, indices, cu, max_s = unpad_input(x, key_padding_mask)
            out = self.forward(x_unpad, cu_seqlens=cu, max_seqlen=max_s)
            return pad_input(out, indices, b, s)
        h, hk, d = self.num_heads, self.num_heads_kv, self.head_dim
        if self.qk_norm is not None:
            return self._forward_qk_norm(x, cu_seqlens, max_seqlen)
        if self.rotary_emb_dim > 0 and cu_seqlens is not None:
            raise NotImplementedError("MHA: rotary embedding with varlen / key_padding_mask input")
        if not self.cross_attn:
            qkv = self.Wqkv(x)
            lead = qkv.shape[:-1]
            if hk == h:
                qkv = qkv.view(*lead, 3, h, d)
                if self.rotary_emb_dim > 0:   # reference mha.py:499-500
                    qkv = self.rotary_emb(qkv)
                context = self.inner_attn(qkv, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen)
            else:
                q = qkv[..., : h * d].reshape(*lead, h, d)
                kv = qkv[..., h * d:].reshape(*lead, 2, hk, d)
                if self.rotary_emb_dim > 0:   # reference mha.py:544-545
                    q, kv = self.rotary_emb(q, kv)
                if cu_seqlens is not None:
                    context = self.inner_cross_attn(q, kv, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen,
                                                    cu_seqlens_k=cu_seqlens, max_seqlen_k=max_seqlen)
                else:
                    context = self.inner_cross_attn(q, kv)
        else:
            assert cu_seqlens is None, "varlen cross attention: call FlashCrossAttention directly"
            x_kv = x if x_kv is None else x_kv
            q = self.Wq(x).reshape(*x.shape[:-1], h, d)
            kv = self.Wkv(x_kv).reshape(*x_kv.shape[:-1], 2, hk, d)
            context = self.inner_cross_attn(q, kv)
        return self.out_proj(context.reshape(*context.shape[:-2], h * d))

    def _split(self, x):
        """q, k, v as (..., heads, head_dim) views of the fused projection."""
        h, hk, d = self.num_heads, self.num_heads_kv, self.head_dim
        qkv = self.Wqkv(x)
        qkv = qkv.view(*qkv.shape[:-1], h + 2 * hk, d)
        return qkv.split((h, hk, hk), dim=-2)

    def _forward_qk_norm(self, x, cu_seqlens, max_seqlen):
        q, k, v = self._split(x)
        dropout_p = self.inner_attn.drop.p if self.training else 0.0
        args = dict(softmax_scale=self.inner_attn.softmax_scale, causal=self.causal)
        if cu_seqlens is None:
            q, k = self.qk_norm(q, k)
            context = flash_attn_func(q, k, v, dropout_p, **args)
        else:
            # rows behind the last sequence get a position like any other: their gradients are zero
            at = torch.arange(x.shape[0], device=x.device, dtype=torch.int32)
            sequence = torch.searchsorted(cu_seqlens[1:], at, right=True).clamp(max=cu_seqlens.numel() - 2)
            positions = (at - cu_seqlens[sequence]).clamp(max=max_seqlen - 1)
            q, k = self.qk_norm(q, k, positions, max_seqlen)
            context = flash_attn_varlen_func(q, k, v, cu_seqlens, cu_seqlens, max_seqlen, max_seqlen, dropout_p, **args)
        return self.out_proj(context.flatten(-2))

    def _forward_cached(self, x, cache, tree_mask, depth):
        if self.cross_attn or not self.causal:
            raise NotImplementedError("MHA: a key/value cache needs causal self-attention")
        if self.rotary_emb_dim > 0 and self.qk_norm is None:
            raise NotImplementedError("MHA: a key/value cache with rotary embedding needs qk_norm=True")
        q, k, v = self._split(x)
        if self.qk_norm is not None:
            if depth is None:
                depth = torch.arange(x.shape[1], device=x.device, dtype=torch.int32)
            q, k = self.qk_norm(q, k, (cache.positions[:, None] + depth).to(torch.int32).expand(x.shape[:2]),
                                cache.most + x.shape[1])
        cache.clear_drafts()
        context = flash_attn_kvcache_func(q, cache.k, cache.v, cache.seqlens, k=k, v=v, block_table=cache.block_table,
                                          tree_mask=tree_mask, softmax_scale=self.inner_attn.softmax_scale,
                                          attn_weight=cache.attn_weight)
        return self.out_proj(context.flatten(-2))
