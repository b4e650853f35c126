"""GPU test of a tree mask that fills its allocation: 64 x 64 tokens are a page of 4 KiB, 2048 x 2048 two segments
of the allocator, with an end of the keys at every kind of place in a step of 128."""
import pytest
import torch

import kvcache_ref as ref
from test_kvcache_gpu import _cache, _check, _need_gpu, _tree   # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("sq,h,hk,lens", [(64, 2, 2, [3, 65]), (64, 8, 2, [64, 100]), (16, 2, 2, [1, 300]), (2048, 1, 1, [1])])
def test_mask_that_ends_with_its_allocation(sq, h, hk, lens):
    from flash_attn import flash_attn_kvcache_func
    torch.manual_seed(0)
    b, d, dtype = len(lens), 64, torch.bfloat16
    lens = torch.tensor(lens, device=DEV, dtype=torch.int32)
    kc, vc, _ = _cache(b, int(lens.max()) + sq, hk, d, dtype, 0)
    q, k, v = (torch.randn(b, sq, n, d, device=DEV).to(dtype) for n in (h, hk, hk))
    mask = _tree(b, sq) if sq < 1000 else torch.rand(b, sq, sq, device=DEV) < 0.5
    kr, vr = kc.clone(), vc.clone()
    out, lse = flash_attn_kvcache_func(q, kc, vc, lens, k, v, tree_mask=mask, return_softmax_lse=True)
    torch.cuda.synchronize()
    _check(out, lse, None, ref.attention(q, kr, vr, lens, k, v, None, mask), dtype, d, 0, 0)
