"""GPU tests of MHA with qk_norm and with a key/value cache: the cached run over a prompt, single tokens
and accepted drafts against the whole sequence at once, and the norm's gradients through the module.

Tolerance: two runs of the same attention differ in the order of their fp32 sums and in which P is rounded
(half a step u of fp16, 2^-11, of each weight: at most u sum p |v| <= u max|v| each), then round
their context (u) and the projection (u, after an fp32 sum over E inputs)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -11


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import flash_attn_2_cuda  # noqa: F401


def _mha(heads, heads_kv, d, rotary, **kw):
    from flash_attn.modules.mha import MHA
    torch.manual_seed(0)
    m = MHA(heads * d, heads, num_heads_kv=heads_kv, causal=True, rotary_emb_dim=rotary, device=DEV, dtype=torch.float16,
            qk_norm=True, **kw)
    with torch.no_grad():
        m.qk_norm.q_weight.uniform_(0.5, 1.5)
        m.qk_norm.k_weight.uniform_(0.5, 1.5)
    return m.eval()


def _bound(m, x, y):
    with torch.no_grad():
        v = m._split(x)[2].float().abs().max()
        w = m.out_proj.weight.float().abs().sum(1)          # each context entry is off by 4 u max|v| at most
        return 4 * U * v * w + 2 * U * y.float().abs()


@pytest.mark.parametrize("heads,heads_kv,d,rotary,inter", [(4, 4, 32, 32, False), (6, 2, 32, 16, True), (4, 1, 96, 0, False)])
def test_cached_run_equals_the_whole_sequence(heads, heads_kv, d, rotary, inter):
    from flash_attn.modules.kv_cache import KVCache
    m = _mha(heads, heads_kv, d, rotary, rotary_emb_interleaved=inter)
    x = torch.randn(3, 60, heads * d, device=DEV, dtype=torch.float16)
    with torch.no_grad():
        whole = m(x)
        cache = KVCache(3, 64, heads_kv, d, device=DEV, dtype=torch.float16)
        parts = []
        for a, b in ((0, 37), (37, 38), (38, 39), (39, 50), (50, 60)):
            parts.append(m(x[:, a:b], kv_cache=cache))
            cache.accept(b - a)
        got = torch.cat(parts, 1)
    assert (got.float() - whole.float()).abs().le(_bound(m, x, whole)).all()
    assert cache.seqlens.tolist() == [60] * 3


def test_tree_commit_and_evict():
    """A path of a drafted tree gives what the same tokens one after another give, and after the commit the
    cache goes on as theirs does; eviction to a budget that everything fits in changes nothing."""
    from flash_attn.modules.kv_cache import KVCache
    heads, d = 4, 32
    m = _mha(heads, 2, d, d)
    x = torch.randn(2, 20, heads * d, device=DEV, dtype=torch.float16)
    drafts = torch.randn(2, 5, heads * d, device=DEV, dtype=torch.float16)
    # tokens 0 - 1 - 3 and 0 - 2 - 4
    parent = [-1, 0, 0, 1, 2]
    mask = torch.zeros(5, 5, dtype=torch.bool)
    for i, p in enumerate(parent):
        if p >= 0:
            mask[i] = mask[p]
        mask[i, i] = True
    mask = mask.to(DEV)
    path = [0, 2, 4]
    with torch.no_grad():
        line, tree = (KVCache(2, 40, 2, d, device=DEV, dtype=torch.float16, track_weight=True) for _ in range(2))
        for c in (line, tree):
            m(x, kv_cache=c)
            c.accept(20)
        y = m(drafts, kv_cache=tree, tree_mask=mask, depth=(mask.sum(1, dtype=torch.int32) - 1))
        accepted = torch.zeros(2, 5, dtype=torch.bool, device=DEV)
        accepted[:, path] = True
        tree.commit(accepted)
        want = m(drafts[:, path], kv_cache=line)
        line.accept(3)
        assert (y[:, path].float() - want.float()).abs().le(_bound(m, torch.cat((x, drafts), 1), want)).all()
        assert torch.equal(tree.seqlens, line.seqlens) and torch.equal(tree.positions, line.positions)
        assert torch.equal(tree.k[:, :23], line.k[:, :23]) and torch.equal(tree.v[:, :23], line.v[:, :23])
        assert (tree.attn_weight[:, :, 23:] == 0).all()
        before = tree.k.clone()
        tree.evict(30)
        assert torch.equal(tree.k, before) and tree.seqlens.tolist() == [23, 23]
        kept = tree.evict(12, sink=2, recent=4)
        assert tree.seqlens.tolist() == [12, 12] and tree.positions.tolist() == [23, 23]
        assert kept[0, 0, :2].tolist() == [0, 1] and kept[0, 0, -4:].tolist() == [19, 20, 21, 22]
        assert torch.isfinite(m(drafts[:, :1], kv_cache=tree)).all()


@pytest.mark.parametrize("varlen", [False, True])
def test_gradients_against_fp64(varlen):
    """The module's gradients against the same computation in fp64 from its parameters: the relative error of
    the norm of each is within 12 half steps (projections, norm, attention and their backward round seven
    times, each relative to the tensor's own size)."""
    heads, hk, d = 4, 2, 32
    m = _mha(heads, hk, d, 16)
    x = torch.randn(1, 50, heads * d, device=DEV, dtype=torch.float16)
    g = torch.randn_like(x)
    lens = [30, 20] if varlen else [50]
    leaf = x.clone().requires_grad_()
    if varlen:
        cu = torch.tensor([0, 30, 50], device=DEV, dtype=torch.int32)
        m(leaf[0], cu_seqlens=cu, max_seqlen=30).backward(g[0])
    else:
        m(leaf).backward(g)
    p = {n: t.detach().double().requires_grad_() for n, t in m.named_parameters()}
    xl = x.double().requires_grad_()
    out = []
    for part in xl[0].split(lens):
        n = part.shape[0]
        qkv = (part @ p["Wqkv.weight"].T + p["Wqkv.bias"]).view(n, heads + 2 * hk, d)
        q, k, v = qkv.split((heads, hk, hk), 1)
        a = torch.outer(torch.arange(n, device=DEV, dtype=torch.float64),
                        10000.0 ** (-torch.arange(0, 16, 2, device=DEV, dtype=torch.float64) / 16))[:, None]

        def norm(t, w):
            z = w * t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6)
            z1, z2 = z[..., :8], z[..., 8:16]
            return torch.cat((z1 * a.cos() - z2 * a.sin(), z1 * a.sin() + z2 * a.cos(), z[..., 16:]), -1)

        q, k = norm(q, p["qk_norm.q_weight"]), norm(k, p["qk_norm.k_weight"])
        k, v = (t.repeat_interleave(heads // hk, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) * d ** -0.5
        s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=DEV).tril(), float("-inf"))
        out.append(torch.einsum("hqk,khd->qhd", s.softmax(-1), v).reshape(n, -1) @ p["out_proj.weight"].T
                   + p["out_proj.bias"])
    torch.cat(out).backward(g[0].double())
    for name, got, want in [("x", leaf.grad, xl.grad)] + [(n, t.grad, p[n].grad) for n, t in m.named_parameters()]:
        err = (got.double() - want).norm() / want.norm()
        assert err <= 12 * U, (name, float(err))


def test_refusals():
    from flash_attn.modules.kv_cache import KVCache
    from flash_attn.modules.mha import MHA
    x = torch.randn(1, 3, 64, device=DEV, dtype=torch.float16)
    cache = KVCache(1, 8, 2, 32, device=DEV, dtype=torch.float16)
    with torch.no_grad():
        for kw, message in ((dict(causal=False), "causal"), (dict(causal=True, rotary_emb_dim=32), "qk_norm")):
            with pytest.raises(NotImplementedError, match=message):
                MHA(64, 2, device=DEV, dtype=torch.float16, **kw)(x, kv_cache=cache)
        with pytest.raises(NotImplementedError, match="inference cache"):
            MHA(64, 2, device=DEV, dtype=torch.float16)(x, inference_params=object())
    with pytest.raises(RuntimeError, match="no backward"):
        MHA(64, 2, causal=True, device=DEV, dtype=torch.float16)(x, kv_cache=cache)
    with pytest.raises(NotImplementedError, match="XPos"):
        MHA(64, 2, qk_norm=True, rotary_emb_dim=32, rotary_emb_scale_base=512)
    with pytest.raises(RuntimeError, match="track_weight"):
        cache.evict(4)


def test_captured_decoding_goes_on():
    """A decoding step with its accept, captured once: each replay stands one token further on."""
    from flash_attn.modules.kv_cache import KVCache
    m = _mha(4, 2, 32, 32)
    x = torch.randn(2, 16, 128, device=DEV, dtype=torch.float16)
    with torch.no_grad():
        whole = m(x)
        cache = KVCache(2, 64, 2, 32, device=DEV, dtype=torch.float16)
        cache.most = 64                            # no position beyond it in any replay
        y = m(x[:, :10], kv_cache=cache)
        cache.accept(10)
        token = x[:, 10:11].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):              # (warm-up: stores the token, without keeping it)
            m(token, kv_cache=cache)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step = m(token, kv_cache=cache)
            cache.accept(1)
        parts = [y]
        for i in range(10, 16):
            token.copy_(x[:, i:i + 1])
            graph.replay()
            parts.append(step.clone())
            torch.cuda.synchronize()
    assert cache.seqlens.tolist() == [16] * 2 and cache.positions.tolist() == [16] * 2
    assert (torch.cat(parts, 1).float() - whole.float()).abs().le(_bound(m, x, whole)).all()
