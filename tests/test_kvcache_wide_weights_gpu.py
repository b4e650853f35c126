"""GPU test of attention weights with more columns than the cache has slots: behind the kept keys 0 up to the last
column, and a sequence whose length is none keeps all of its own."""
import pytest
import torch

from test_kvcache_gpu import _cache, _need_gpu   # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("page", [0, 16])
def test_evict_with_more_columns_than_slots(page):
    from flash_attn import flash_attn_kvcache_evict_
    kc, vc, table = _cache(4, 64, 2, 64, torch.float16, page)
    w = torch.rand(4, 2, 75, device=DEV) + 1
    lens = torch.tensor([64, 9, 65, -1], device=DEV, dtype=torch.int32)
    want_k = kc.clone(), vc.clone()
    ref = flash_attn_kvcache_evict_(*want_k, lens, w[:, :, :64], 20, sink=2, recent=3, block_table=table)
    new, got, kept = flash_attn_kvcache_evict_(kc, vc, lens, w, 20, sink=2, recent=3, block_table=table)
    assert new.tolist() == [20, 9, 65, -1] and torch.equal(new, ref[0]) and torch.equal(kept, ref[2])
    assert torch.equal(kc, want_k[0]) and torch.equal(vc, want_k[1]) and torch.equal(got[:, :, :64], ref[1])
    assert (got[:2, :, 64:] == 0).all() and torch.equal(got[2:], w[2:])
