"""CPU tests of sizes near 2^31 and of the workspace: what the cache operators refuse and ask for."""
import pytest
import torch

BF = torch.bfloat16


def _cache():
    return (torch.zeros(1, 50, 2, 64, dtype=BF), torch.zeros(1, 50, 2, 64, dtype=BF), torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("budget", [2 ** 31 - 1, 2 ** 31 - 300, 0x7fff0001])
def test_budgets_that_the_counters_would_run_over(budget):
    """The kernel's threads go over the budget's places 1024 apart in 32-bit counters."""
    from flash_attn import flash_attn_kvcache_evict_
    with pytest.raises(RuntimeError, match="budget"):
        flash_attn_kvcache_evict_(*_cache(), torch.zeros(1, 2, 50), budget)


def test_slots_that_the_counters_would_run_over():
    """A table of few, large pages (the same one over and over) names more keys than there is memory."""
    from flash_attn import flash_attn_kvcache_evict_, flash_attn_kvcache_func
    k, v, lens = torch.empty(1, 1 << 15, 1, 8, dtype=BF), torch.empty(1, 1 << 15, 1, 8, dtype=BF), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 1, 8, dtype=BF)
    for blocks, message in (((1 << 16) - 1, "too many slots"), ((1 << 16) - 2, "on the GPU")):
        table = torch.zeros(1, blocks, dtype=torch.int32)
        with pytest.raises(RuntimeError, match=message):
            flash_attn_kvcache_func(q, k, v, lens, block_table=table)
    with pytest.raises(RuntimeError, match="too many slots"):
        flash_attn_kvcache_evict_(k, v, lens, torch.zeros(1, 1, 50), 10, block_table=torch.zeros(1, (1 << 16) - 1, dtype=torch.int32))


def test_a_prompt_needs_no_workspace():
    """Row tiles that fill the chip by themselves walk all keys: no sequence is cut, nothing is left to merge."""
    import ctypes
    import flash_attn_2_cuda as m
    w = m._lib.flash_attn_kvcache_workspace
    w.argtypes, w.restype = [ctypes.c_int] * 6 + [ctypes.c_bool], ctypes.c_size_t
    assert w(1, 8192, 16384, 32, 8, 128, False) == 0
    assert w(4, 4096, 4096, 64, 64, 64, True) == 0
    assert w(1, 48, 16384, 32, 8, 128, False) > 0   # a tree is cut


@pytest.mark.gpu
@pytest.mark.parametrize("d,weight", [(64, False), (128, True)])
def test_a_prompt_that_is_not_cut(d, weight):
    """Enough heads and tokens for one share: every sequence is written at once, weights included."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import flash_attn_2_cuda as m
    from test_kvcache_gpu import _run
    assert m._lib.flash_attn_kvcache_workspace(2, 1100, 1200, 256, 256, d, weight) == 0
    _run(2, 1100, 256, 256, d, [0, 37], torch.bfloat16, 0, weight=weight, slack=63)
