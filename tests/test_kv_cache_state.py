"""The state of a KVCache over calls (flash_attn.modules.kv_cache)."""
import pytest
import torch

from flash_attn.modules.kv_cache import KVCache


def test_most_stops_at_the_longest_position():
    c = KVCache(2, 100, 1, 8, max_position=50)
    for _ in range(3):
        c.accept(15)
    assert c.most == 45
    c.accept(15)
    assert c.most == 50
    c = KVCache(2, 100, 1, 8)
    c.accept(70)
    assert c.most == 70


@pytest.mark.gpu
def test_commits_of_large_trees_do_not_grow_the_table():
    """64 drafted tokens a step of which one stays: positions reach 40, and the table does not grow past the
    longest position and a call's tokens."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from flash_attn.modules.mha import MHA
    torch.manual_seed(0)
    m = MHA(64, 2, causal=True, rotary_emb_dim=32, qk_norm=True, device="cuda", dtype=torch.float16)
    caches = [KVCache(1, 128, 2, 32, device="cuda", dtype=torch.float16, max_position=n) for n in (64, None)]
    accepted = torch.zeros(1, 64, dtype=torch.bool, device="cuda")
    accepted[0, 0] = True
    rows = []
    with torch.no_grad():
        for c in caches:
            m.qk_norm._tables.clear()
            for step in range(40):
                torch.manual_seed(step)
                y = m(torch.randn(1, 64, 64, device="cuda", dtype=torch.float16), kv_cache=c)
                c.commit(accepted)
            rows.append((m.qk_norm.table(1, "cuda")[0].shape[0], y))
    assert rows[0][0] == 128 and rows[1][0] >= 40 * 64
    assert torch.equal(rows[0][1], rows[1][1]) and caches[0].positions.tolist() == [40]
