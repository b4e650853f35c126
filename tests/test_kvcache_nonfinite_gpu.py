"""GPU test of infinities and NaN in V: a cached key's reach every row, wherever the key lies in a step and whatever
drafted keys lie beside it, and no other column changes."""
import pytest
import torch

import kvcache_ref as ref
from test_kvcache_gpu import _cache, _need_gpu, _tree   # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("page", [0, 17, 32])
@pytest.mark.parametrize("sq,h", [(1, 2), (6, 2), (24, 4), (40, 4)])   # row tiles of 32, 64 and 128
@pytest.mark.parametrize("new", [True, False])
def test_cached_values_reach_every_row(new, sq, h, page):
    from flash_attn import flash_attn_kvcache_func
    torch.manual_seed(0)
    b, hk, d, n = 1, 2, 64, 40             # keys 32 .. 39 share their 32 with the first drafted ones
    lens = torch.tensor([n], device=DEV, dtype=torch.int32)
    kc, vc, table = _cache(b, n + sq, hk, d, torch.float16, page)
    # (scores near zero: no weight of a key rounds to zero, and infinity stays what it is)
    q = 0.1 * torch.randn(b, sq, h, d, device=DEV).half()
    k, v = (torch.randn(b, sq, hk, d, device=DEV).half() for _ in range(2))
    args = (lens, k, v) if new else (lens, None, None)
    clean = flash_attn_kvcache_func(q, kc.clone(), vc.clone(), *args, block_table=table)
    for r in range(n):
        bad = vc.clone()
        at = ref.slot(kc, table, 0, torch.tensor([r], device=DEV))
        bad[at[0], at[1], 0, 5], bad[at[0], at[1], 1, 8] = float("inf"), float("nan")
        out = flash_attn_kvcache_func(q, kc.clone(), bad, *args, block_table=table)
        want = clean.clone()
        want[:, :, :h // 2, 5], want[:, :, h // 2:, 8] = float("inf"), float("nan")
        torch.testing.assert_close(out, want, rtol=0, atol=0, equal_nan=True, msg=lambda m: f"key {r}: {m}")


@pytest.mark.parametrize("sq", [5, 40])
def test_cached_and_drafted_values_in_one_step(sq):
    """Both in the same 32 keys: the cached one reaches all rows, the drafted one those that see it."""
    from flash_attn import flash_attn_kvcache_func
    torch.manual_seed(0)
    n, hk, d = 43, 2, 128
    lens = torch.tensor([n], device=DEV, dtype=torch.int32)
    mask = _tree(1, sq)
    kc, vc, _ = _cache(1, n + sq, hk, d, torch.float16, 0)
    q = 0.1 * torch.randn(1, sq, hk, d, device=DEV).half()
    k, v = (torch.randn(1, sq, hk, d, device=DEV).half() for _ in range(2))
    clean = flash_attn_kvcache_func(q, kc.clone(), vc.clone(), lens, k, v, tree_mask=mask)
    vc[0, n - 2, :, 7] = float("-inf")
    v[0, 1, :, 7], v[0, 1, :, 100] = float("inf"), float("nan")
    out = flash_attn_kvcache_func(q, kc, vc, lens, k, v, tree_mask=mask)
    see = mask[0, :, 1][:, None].expand(sq, hk)
    want = clean.clone()
    want[0, :, :, 7] = torch.where(see, float("nan"), float("-inf"))
    want[0, :, :, 100] = torch.where(see, float("nan"), clean[0, :, :, 100].float())
    torch.testing.assert_close(out, want, rtol=0, atol=0, equal_nan=True)
    assert see.any() and not see.all()


@pytest.mark.parametrize("sq", [4, 40])
@pytest.mark.parametrize("new", [True, False])
@pytest.mark.parametrize("n", [3, 1000])
def test_a_weight_of_zero_makes_infinity_nan(n, new, sq):
    """A drafted key that a row sees with a weight that is zero in fp32 (2^-1000 of the largest): 0 x inf."""
    from flash_attn import flash_attn_kvcache_func
    torch.manual_seed(0)
    hk, d = 2, 64
    lens = torch.tensor([n], device=DEV, dtype=torch.int32)
    kc, vc, _ = _cache(1, n + sq, hk, d, torch.float16, 0)
    q = torch.zeros(1, sq, hk, d, device=DEV, dtype=torch.float16)
    k, v = (torch.randn(1, sq, hk, d, device=DEV).half() for _ in range(2))
    q[..., 0], kc[..., 0], k[..., 0] = 8, 0, 0
    k[0, 1, 0, 0] = -700                   # head 0: score -8 x 700 / 8 = -700 against 0; head 1: 0
    v[0, 1, :, 9] = float("inf")
    if not new:
        kc[0, n:], vc[0, n:] = k[0], v[0]
    out, lse = flash_attn_kvcache_func(q, kc, vc, lens, *((k, v) if new else ()), return_softmax_lse=True)
    assert torch.isfinite(lse).all() and torch.isfinite(out[..., :9]).all() and torch.isfinite(out[0, 0]).all()
    assert torch.isnan(out[0, 1:, 0, 9]).all() and torch.isposinf(out[0, 1:, 1, 9]).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_many_nonfinite_drafts_do_not_hold_the_gpu(value, d):
    """A prompt with a V channel that overflowed in every token: what is taken out and added again one key after
    another stays a matter of milliseconds."""
    from flash_attn import flash_attn_kvcache_func
    torch.manual_seed(0)
    sq, h, hk = 1024, 4, 2
    lens = torch.tensor([5], device=DEV, dtype=torch.int32)
    kc, vc, _ = _cache(1, 5 + sq, hk, d, torch.float16, 0)
    q = 0.1 * torch.randn(1, sq, h, d, device=DEV).half()
    k, v = (torch.randn(1, sq, hk, d, device=DEV).half() for _ in range(2))
    clean = flash_attn_kvcache_func(q, kc, vc, lens, k, v)
    v[..., 3], v[:, :, 1, 40:] = value, value
    times = []
    for _ in range(2):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        out = flash_attn_kvcache_func(q, kc, vc, lens, k, v)
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end))
    assert min(times) < 200, times
    want = clean.clone()
    want[..., 3], want[:, :, h // 2:, 40:] = value, value
    torch.testing.assert_close(out, want, rtol=0, atol=0, equal_nan=True)
