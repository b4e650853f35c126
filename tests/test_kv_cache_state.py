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


def test_clear_drafts_leaves_the_keys_held():
    c = KVCache(3, 10, 2, 8, track_weight=True)
    c.attn_weight.uniform_(1, 2)
    before = c.attn_weight.clone()
    c.seqlens.copy_(torch.tensor([0, 4, 10], dtype=torch.int32))
    c.clear_drafts()
    for i, n in enumerate((0, 4, 10)):
        assert torch.equal(c.attn_weight[i, :, :n], before[i, :, :n]) and (c.attn_weight[i, :, n:] == 0).all()
    KVCache(3, 10, 2, 8).clear_drafts()            # nothing tracked: nothing to clear


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_tokens_that_were_not_kept_leave_no_weight(captured):
    """A rejected draft (or the warm-up of a capture), then a token that stays: its slot's weight is its own."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from flash_attn.modules.mha import MHA
    torch.manual_seed(0)
    m = MHA(64, 2, causal=True, device="cuda", dtype=torch.float16)
    x = torch.randn(2, 13, 64, device="cuda", dtype=torch.float16)
    with torch.no_grad():
        a, b = (KVCache(2, 32, 2, 32, device="cuda", dtype=torch.float16, track_weight=True) for _ in range(2))
        for c in (a, b):
            m(x[:, :10], kv_cache=c)
            c.accept(10)
        if captured:
            token = x[:, :1].clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                m(token, kv_cache=a)               # warm-up: not kept
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                m(token, kv_cache=a)
                a.accept(1)
            m(x[:, 5:8], kv_cache=a)               # eager between the replays, not kept either
            for i in (10, 11, 12):
                token.copy_(x[:, i:i + 1])
                graph.replay()
                torch.cuda.synchronize()
        else:
            m(x[:, :3], kv_cache=a)
            for i in (10, 11, 12):
                m(x[:, i:i + 1], kv_cache=a)
                a.accept(1)
        for i in (10, 11, 12):
            m(x[:, i:i + 1], kv_cache=b)
            b.accept(1)
    assert (b.attn_weight[:, :, 10:13] > 0).all()
    if not captured:
        assert torch.equal(a.attn_weight[:, :, 10:], b.attn_weight[:, :, 10:])
    else:
        # The graph projects from `token`, contiguous, the other run from a slice of x: the library may sum the two
        # products in another order, so that entries of q and k differ by a rounding step, 2 u relative (u = 2^-11).
        # A score sum q k / sqrt(d) then differs by ds <= 4 u sum |q k| / sqrt(d) <= 4 u |q| |k| / sqrt(d), a
        # probability by the factor exp(+- 2 ds), and a weight, a sum of them, likewise.
        q, k, _ = m._split(x)
        ds = 4 * 2.0 ** -11 * float(q.float().norm(dim=-1).max() * k.float().norm(dim=-1).max()) / 32 ** 0.5
        assert ds < 0.02
        err = (a.attn_weight[:, :, 10:] - b.attn_weight[:, :, 10:]).abs()
        assert (err <= 1.03 * 2 * ds * b.attn_weight[:, :, 10:]).all()
    assert a.seqlens.tolist() == [13, 13] and (a.attn_weight[:, :, 13:] == 0).all()


@pytest.mark.parametrize("paged", [False, True])
def test_accept_leaves_a_sequence_without_room(paged):
    """The call stored nothing for it: its length stays one that eviction and commit take."""
    c = KVCache(3, 8 if paged else 32, 1, 8)
    if paged:
        c.block_table = torch.zeros(3, 4, dtype=torch.int32)
    c.seqlens.copy_(torch.tensor([0, 28, 29], dtype=torch.int32))
    c.positions.copy_(torch.tensor([0, 50, 51], dtype=torch.int32))
    c.accept(4)
    assert c.seqlens.tolist() == [4, 32, 29] and c.positions.tolist() == [4, 54, 51]
    assert c.seqlens.dtype == c.positions.dtype == torch.int32
    c.attn_weight = torch.zeros(3, 1, 10)          # fewer columns than slots
    c.accept(6)
    assert c.seqlens.tolist() == [10, 32, 29]


@pytest.mark.gpu
def test_a_full_cache_goes_on_after_eviction():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from flash_attn.modules.mha import MHA
    torch.manual_seed(0)
    m = MHA(64, 2, causal=True, device="cuda", dtype=torch.float16)
    x = torch.randn(2, 16, 64, device="cuda", dtype=torch.float16)
    with torch.no_grad():
        c = KVCache(2, 16, 2, 32, device="cuda", dtype=torch.float16, track_weight=True)
        m(x[:, :15], kv_cache=c)
        c.accept(15)
        assert torch.isnan(m(x[:, :3], kv_cache=c)).all()
        c.accept(3)                                # nothing was stored
        assert c.seqlens.tolist() == [15, 15]
        kept = c.evict(8, sink=2, recent=2)
        assert c.seqlens.tolist() == [8, 8] and (kept >= 0).all()
        assert torch.isfinite(m(x[:, :3], kv_cache=c)).all()
        c.accept(3)
        assert c.seqlens.tolist() == [11, 11] and c.positions.tolist() == [18, 18]


@pytest.mark.parametrize("columns", [10, 6, 14])
def test_clear_drafts_of_weights_that_were_put_in(columns):
    c = KVCache(2, 10, 2, 8)
    c.attn_weight = torch.ones(2, 2, columns)
    c.seqlens.copy_(torch.tensor([3, 6], dtype=torch.int32))
    c.clear_drafts()
    assert c.attn_weight.sum(-1).tolist() == [[3, 3], [6, 6]]
