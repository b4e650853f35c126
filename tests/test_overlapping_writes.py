"""CPU tests of written tensors that are views of one tensor: refused when they share an element, however their
heads, rows or sequences overlap, and taken when they only interleave."""
import pytest
import torch

from flash_attn import flash_attn_kvcache_commit_
from flash_attn.layers.qk_norm import apply_qk_norm_rotary_func

BF = torch.bfloat16


def _inplace(q, k):
    with torch.no_grad():
        apply_qk_norm_rotary_func(q, k, inplace=True)


def test_views_that_share_elements_are_refused():
    x = torch.zeros(4, 10, 12, 64, dtype=BF)
    y = torch.zeros(2, 24, 6, 64, dtype=BF)
    for q, k in ((x[:, :, :4], x[:, :, 3:6]), (x[:, :, 3:6], x[:, :, :4]),
                 (x[:2, :, :4], x[1:3, :, 2:3]), (x[:, :5, :4], x[:, 4:9, :4]), (x[..., :32], x[..., 16:48]),
                 (y[:, :12], y[:, 6:18]), (x[:1, :, :1], x[:1, :, :1])):
        with pytest.raises(RuntimeError, match="share memory"):
            _inplace(q, k)


def test_views_that_interleave_are_taken():
    x = torch.zeros(4, 10, 12, 64, dtype=BF)
    for q, k in ((x[:, :, :4], x[:, :, 4:6]), (x[:, :, ::2], x[:, :, 1::2]), (x[:2, :, :4], x[2:, :, :4]),
                 (x[:, :5, :4], x[:, 5:, 2:4]), (x[:, ::2], x[:, 1::2]), (x[..., :32], x[..., 32:]),
                 (x[:1, :, :3], x[1:2, :, :5])):
        with pytest.raises(RuntimeError, match="on the GPU"):
            _inplace(q, k)
    kv = torch.zeros(2, 30, 2, 4, 64, dtype=BF)
    lens, accepted = torch.zeros(2, dtype=torch.int32), torch.ones(2, 3, dtype=torch.bool)
    with pytest.raises(RuntimeError, match="on the GPU"):
        flash_attn_kvcache_commit_(kv[:, :, 0], kv[:, :, 1], lens, accepted)
    flat = torch.zeros(2, 35, 4, 64, dtype=BF)
    with pytest.raises(RuntimeError, match="share memory"):
        flash_attn_kvcache_commit_(flat[:, :30], flat[:, 5:], lens, accepted)
