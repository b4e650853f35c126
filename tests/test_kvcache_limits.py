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
