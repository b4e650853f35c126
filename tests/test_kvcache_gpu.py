"""GPU tests of the key/value cache operators (csrc/fa_kvcache.hip, fa_evict.hip) against tests/kvcache_ref.py
in fp64.

Tolerances of the attention, with u = eps / 2 of the type (half a step), ds = d 2^-24 max sum |q k| scale
(fp32 accumulation of a score) and w = 2 ds + 2^-19 (what that and the fp32 exponentials, sums and
merges make of a probability, relatively):
  out: u |out| (its own rounding) + (u + w) sum p |v| (P is rounded to the type for its product), and
       for fp16 2^-25 sum |v| (P below its normal range);
  lse: w (1 + |lse|);     weight: w times the mass (fp32 throughout).
Moves are compared bit for bit."""
import pytest
import torch

import kvcache_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import flash_attn_2_cuda  # noqa: F401


def _cache(b, slots, hk, d, dtype, page, seed=0, fill=None):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    if page:
        blocks = -(-slots // page)
        shape = (b * blocks + 2, page, hk, d)
        table = torch.randperm(b * blocks + 2, generator=g, device=DEV)[:b * blocks].to(torch.int32).reshape(b, blocks)
    else:
        shape, table = (b, slots, hk, d), None
    return [torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2)] + [table]


def _tree(b, sq, seed=0):
    g = torch.Generator().manual_seed(seed)
    m = torch.zeros(b, sq, sq, dtype=torch.bool)
    for x in range(b):
        for i in range(sq):
            if i:
                m[x, i] = m[x, int(torch.randint(0, i, (1,), generator=g))]
            m[x, i, i] = True
    return m.to(DEV)


def _close(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol) & ~(got.double() == want)
    assert not bad.any(), (what, int(bad.sum()), float(err[bad].max()), float((err / tol)[bad].max()))


def _check(out, lse, weight, r, dtype, d, vmax, keys):
    want, wlse, wweight, mass, score = r
    u = torch.finfo(dtype).eps / 2
    ds = d * 2.0 ** -24 * score
    w = 2 * ds + 2.0 ** -19
    tol = u * want.abs() + (u + w.transpose(1, 2)[..., None]) * mass
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25 * vmax * keys
    _close(out, want, tol, "out")
    _close(lse, wlse, w * (1 + torch.where(torch.isinf(wlse), 0.0, wlse).abs()), "lse")
    if weight is not None:
        _close(weight, wweight, float(w.max()) * wweight.abs() + 1e-30, "weight")


def _run(b, sq, h, hk, d, lens, dtype, page=0, tree=False, new=True, weight=True, slack=5, scale=None, seed=0):
    from flash_attn import flash_attn_kvcache_func
    torch.manual_seed(seed)
    lens = torch.tensor(lens, device=DEV, dtype=torch.int32)
    slots = int(lens.max()) + sq + slack
    kc, vc, table = _cache(b, slots, hk, d, dtype, page, seed)
    slots = slots if table is None else table.shape[1] * page
    # nothing behind a sequence is read: NaN there
    for i, n in enumerate(lens.tolist()):
        j = torch.arange(n + (0 if new else sq), slots, device=DEV)
        at = ref.slot(kc, table, i, j)
        kc[at], vc[at] = float("nan"), float("nan")
    q = torch.randn(b, sq, h, d, device=DEV).to(dtype)
    k, v = (torch.randn(b, sq, hk, d, device=DEV).to(dtype) if new else None for _ in range(2))
    mask = _tree(b, sq, seed) if tree else None
    kr, vr = kc.clone(), vc.clone()
    acc = torch.rand(b, hk, slots, device=DEV) if weight else None
    before = acc.clone() if weight else None
    out, lse = flash_attn_kvcache_func(q, kc, vc, lens, k=k, v=v, block_table=table, tree_mask=mask,
                                       softmax_scale=scale, attn_weight=acc, return_softmax_lse=True)
    torch.cuda.synchronize()
    r = ref.attention(q, kr, vr, lens, k, v, table, mask, scale)
    assert torch.equal(kc.view(torch.int16), kr.view(torch.int16)) and torch.equal(vc.view(torch.int16), vr.view(torch.int16))
    _check(out, lse, None, r, dtype, d, float(vr[~torch.isnan(vr)].abs().max()), int(lens.max()) + sq)
    if weight:
        # the sum's own rounding (2^-24 of it) on top of the mass's
        w = 2 * d * 2.0 ** -24 * float(r[4].max()) + 2.0 ** -19
        want = before.double() + r[2]
        _close(acc, want, 2.0 ** -23 * want.abs() + w * r[2], "weight")
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [8, 40, 64, 96, 128, 136, 256])
@pytest.mark.parametrize("page", [0, 1, 17, 64])
def test_decode(page, d, dtype):
    _run(4, 1, 8, 2, d, [0, 1, 127, 700], dtype, page)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sq,h,hk", [(2, 3, 3), (13, 4, 4), (7, 12, 3), (48, 8, 2), (33, 2, 1), (64, 16, 2), (5, 7, 1),
                                     (130, 2, 2), (9, 128, 1)])
@pytest.mark.parametrize("d,page", [(128, 0), (64, 16), (192, 40)])
def test_tree(d, page, sq, h, hk, dtype):
    _run(3, sq, h, hk, d, [0, 333, 130], dtype, page, tree=True)


@pytest.mark.parametrize("sq", [1, 4, 40])
@pytest.mark.parametrize("n", [0, 1, 31, 32, 33, 127, 128, 129, 255, 256, 1023, 5000])
def test_lengths(n, sq):
    _run(1, sq, 4, 1, 64, [n], torch.bfloat16, 0)


@pytest.mark.parametrize("page", [0, 32])
def test_drafts_already_in_the_cache(page):
    _run(2, 6, 8, 4, 128, [77, 200], torch.bfloat16, page, tree=True, new=False)


def test_long_and_full_cache():
    _run(2, 3, 8, 2, 128, [70001, 12345], torch.bfloat16, 0, slack=0)
    _run(1, 20, 16, 2, 128, [40000], torch.float16, 256, tree=True, slack=0)


def test_scale_and_large_scores():
    _run(2, 5, 4, 2, 64, [50, 300], torch.float16, 0, tree=True, scale=0.7)
    _run(2, 1, 4, 2, 64, [50, 300], torch.bfloat16, 0, scale=2.0)


def test_rows_that_see_nothing_and_masked_garbage():
    """An empty mask row on an empty cache gives 0 and +inf; drafts that nobody sees may hold NaN."""
    from flash_attn import flash_attn_kvcache_func
    b, sq, hk, d = 2, 6, 2, 64
    kc, vc, _ = _cache(b, 300, hk, d, torch.bfloat16, 0)
    lens = torch.tensor([0, 200], device=DEV, dtype=torch.int32)
    mask = _tree(b, sq)
    mask[:, :, 3] = False          # nobody sees draft 3
    mask[:, 4] = False             # draft 4 sees no draft
    q = torch.randn(b, sq, 4, d, device=DEV, dtype=torch.bfloat16)
    k, v = torch.randn(b, sq, hk, d, device=DEV, dtype=torch.bfloat16), torch.randn(b, sq, hk, d, device=DEV, dtype=torch.bfloat16)
    k[:, 3], v[:, 3] = float("nan"), float("inf")
    w = torch.zeros(b, hk, 300, device=DEV)
    kr, vr = kc.clone(), vc.clone()
    out, lse = flash_attn_kvcache_func(q, kc, vc, lens, k, v, tree_mask=mask, attn_weight=w, return_softmax_lse=True)
    r = ref.attention(q, kr, vr, lens, k, v, None, mask)
    _check(out, lse, w, r, torch.bfloat16, d, 0, 0)
    assert (out[0, 4] == 0).all() and torch.isposinf(lse[0, :, 4]).all()
    assert torch.isfinite(out).all() and (w[:, :, 3][0] == 0).all()


@pytest.mark.parametrize("sq,d,n", [(6, 64, 40), (40, 128, 300), (3, 256, 0), (70, 128, 1000)])
@pytest.mark.parametrize("new", [True, False])
def test_nonfinite_values_reach_only_the_rows_that_see_them(new, sq, d, n):
    from flash_attn import flash_attn_kvcache_func
    b, hk = 2, 2
    lens = torch.tensor([n, n + 7], device=DEV, dtype=torch.int32)
    mask = _tree(b, sq)
    kc, vc, _ = _cache(b, n + 7 + sq, hk, d, torch.float16, 0)
    q, k, v = (torch.randn(b, sq, hk, d, device=DEV, dtype=torch.float16) for _ in range(3))
    bad = sq - 2
    v[:, bad, 0, 5], v[:, bad, 1, 8] = float("inf"), float("nan")
    if not new:
        for i in range(b):
            at = int(lens[i])
            kc[i, at:at + sq], vc[i, at:at + sq] = k[i], v[i]
    out = flash_attn_kvcache_func(q, kc.clone(), vc.clone(), lens, *((k, v) if new else ()), tree_mask=mask)
    v0 = torch.where(torch.isfinite(v), v, 0.0)
    if not new:
        vc = torch.where(torch.isfinite(vc), vc, 0.0)
    clean = flash_attn_kvcache_func(q, kc, vc, lens, *((k, v0) if new else ()), tree_mask=mask)
    see = mask[:, :, bad]
    want = clean.clone()
    want[:, :, 0, 5] = torch.where(see, float("inf"), clean[:, :, 0, 5])
    want[:, :, 1, 8] = torch.where(see, float("nan"), clean[:, :, 1, 8])
    torch.testing.assert_close(out, want, rtol=0, atol=0, equal_nan=True)
    assert not see.all()


def test_lengths_without_room_and_bad_pages():
    from flash_attn import flash_attn_kvcache_func
    kc, vc, _ = _cache(4, 64, 2, 64, torch.float16, 0)
    q = torch.randn(4, 3, 4, 64, device=DEV, dtype=torch.float16)
    k = torch.randn(4, 3, 2, 64, device=DEV, dtype=torch.float16)
    lens = torch.tensor([62, 10, -1, 2 ** 31 - 1], device=DEV, dtype=torch.int32)
    before, w = kc.clone(), torch.zeros(4, 2, 64, device=DEV)
    out, lse = flash_attn_kvcache_func(q, kc, vc, lens, k, k, attn_weight=w, return_softmax_lse=True)
    assert torch.isnan(out[[0, 2, 3]]).all() and torch.isnan(lse[[0, 2, 3]]).all()
    assert torch.isfinite(out[1]).all()
    assert torch.equal(kc[[0, 2, 3]], before[[0, 2, 3]]) and (w[[0, 2, 3]] == 0).all()
    assert torch.equal(kc[1, 10:13], k[1])
    for sq in (1, 40):
        kc, vc, table = _cache(3, 200, 2, 64, torch.float16, 16)
        q = torch.randn(3, sq, 4, 64, device=DEV, dtype=torch.float16)
        k = torch.randn(3, sq, 2, 64, device=DEV, dtype=torch.float16)
        table[1, 3], table[2, 0] = kc.shape[0], -5
        lens = torch.tensor([100, 100, 100], device=DEV, dtype=torch.int32)
        out = flash_attn_kvcache_func(q, kc, vc, lens, k, k, block_table=table)
        assert torch.isfinite(out[0]).all() and torch.isnan(out[1:]).all()
        lens = torch.tensor([40, 40, 40], device=DEV, dtype=torch.int32)   # page 3 of sequence 1 is not reached
        out = flash_attn_kvcache_func(q[:, :1], kc, vc, lens, k[:, :1], k[:, :1], block_table=table)
        assert torch.isfinite(out[:2]).all() and torch.isnan(out[2]).all()


def test_strides_and_views():
    """q, k, v as views of one projection, caches as halves of a packed one, a mask without batch."""
    from flash_attn import flash_attn_kvcache_func
    b, sq, h, hk, d = 2, 5, 6, 2, 128
    qkv = torch.randn(b, sq, h + 2 * hk, d, device=DEV, dtype=torch.bfloat16)
    kv = torch.randn(b, 90, 2, hk, d, device=DEV, dtype=torch.bfloat16)
    kc, vc = kv[:, :, 0], kv[:, :, 1]
    lens = torch.tensor([80, 3], device=DEV, dtype=torch.int32)
    mask = _tree(1, sq)[0]
    kr, vr = kc.clone(), vc.clone()
    q, k, v = qkv[:, :, :h], qkv[:, :, h:h + hk], qkv[:, :, h + hk:]
    out, lse = flash_attn_kvcache_func(q, kc, vc, lens, k, v, tree_mask=mask, return_softmax_lse=True)
    r = ref.attention(q, kr, vr, lens, k, v, None, mask)
    _check(out, lse, None, r, torch.bfloat16, d, 0, 0)
    assert torch.equal(kc, kr) and torch.equal(vc, vr)
    # an unaligned q is copied; a transposed mask too
    q2 = torch.randn(b, sq, h, d + 3, device=DEV, dtype=torch.bfloat16)[..., 3:]
    mt = mask.t().contiguous().t()
    out = flash_attn_kvcache_func(q2, kc, vc, lens, k, v, tree_mask=mt)
    assert torch.equal(out, flash_attn_kvcache_func(q2.contiguous(), kc, vc, lens, k, v, tree_mask=mask))


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements: the last sequence's keys lie behind them."""
    from flash_attn import flash_attn_kvcache_commit_, flash_attn_kvcache_evict_, flash_attn_kvcache_func
    slots, hk, d = 1100000, 8, 128
    kc, vc = (torch.empty(2, slots, hk, d, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    assert kc.numel() > 2 ** 31
    n = slots - 3
    small = torch.randn(2, 700, hk, d, device=DEV, dtype=torch.bfloat16)
    kc[1, :].zero_(); vc[1, :].zero_()
    kc[1, n - 700:n], vc[1, n - 700:n] = small[0], small[1]
    lens = torch.tensor([0, n], device=DEV, dtype=torch.int32)
    q, k, v = (torch.randn(2, 2, hk, d, device=DEV, dtype=torch.bfloat16) * 4 for _ in range(3))
    out = flash_attn_kvcache_func(q, kc, vc, lens, k, v)
    keys, vals = (torch.cat((small[i], x[1])).double() for i, x in ((0, k), (1, v)))
    for head in range(hk):
        s = q[1, :, head].double() @ keys[:, head].T * d ** -0.5
        s[0, -1] = float("-inf")
        s = torch.cat((torch.zeros(2, n - 700, device=DEV, dtype=torch.float64), s), 1)
        p = torch.softmax(s, 1)[:, n - 700:]
        want = p @ vals[:, head]
        tol = 2.0 ** -9 * want.abs() + 2.0 ** -8 * (p @ vals[:, head].abs()) + 1e-6
        assert ((out[1, :, head].double() - want).abs() <= tol).all()
    assert torch.equal(kc[1, n:n + 2], k[1])
    acc = torch.tensor([[False, True]], device=DEV).expand(2, 2)
    new = flash_attn_kvcache_commit_(kc, vc, lens, acc)
    assert new.tolist() == [1, n + 1] and torch.equal(kc[1, n], k[1, 1])
    w = torch.zeros(2, hk, slots, device=DEV)
    w[1, :, n - 700:n:7] = 1.0
    new, _, kept = flash_attn_kvcache_evict_(kc, vc, new, w, 200, sink=1, recent=1)
    want = [0] + list(range(1, 1 + 98)) + list(range(n - 700, n, 7)) + [n]
    assert new.tolist() == [1, 200] and kept[1, 3].tolist() == want
    assert torch.equal(kc[1, 99:199], small[0][::7]) and torch.equal(vc[1, 199], v[1, 1])
    del kc, vc, w
    torch.cuda.empty_cache()


@pytest.mark.parametrize("page", [0, 1, 24])
@pytest.mark.parametrize("hk,d,lens,budget,sink,recent", [
    (2, 64, [100, 40, 41, 0], 40, 4, 10), (1, 128, [5000], 1200, 0, 0), (3, 8, [65, 300], 64, 0, 64),
    (2, 256, [700, 699], 130, 100, 30), (1, 40, [33], 1, 0, 0), (1, 40, [33], 1, 1, 0), (4, 96, [2500, 9], 2499, 7, 11),
    (2, 128, [1500, 20], 3000, 1, 1), (2, 8, [20000, 9000], 8888, 5, 100), (1, 16, [70000], 30000, 0, 1)])
def test_evict(hk, d, lens, budget, sink, recent, page):
    from flash_attn import flash_attn_kvcache_evict_
    b = len(lens)
    lens = torch.tensor(lens, device=DEV, dtype=torch.int32)
    kc, vc, table = _cache(b, int(lens.max()) + 3, hk, d, torch.float16, page)
    slots = kc.shape[1] * (1 if table is None else table.shape[1])
    w = torch.exp(torch.randn(b, hk, slots, device=DEV))
    w[:, :, ::5] = 0.0                        # ties
    w[:, :, 3::11] = 0.25
    kr, vr, keep = kc.clone(), vc.clone(), w.clone()
    got = flash_attn_kvcache_evict_(kc, vc, lens, w, budget, sink=sink, recent=recent, block_table=table)
    want = ref.evict(kr, vr, lens, w, budget, sink, recent, table)
    assert torch.equal(w, keep)
    for a, x in zip(got, want):
        assert torch.equal(a, x)
    assert torch.equal(kc, kr) and torch.equal(vc, vr)


def test_evict_odd_weights():
    """All equal, all zero of both signs, infinities, negatives, NaN (heaviest) and denormals."""
    from flash_attn import flash_attn_kvcache_evict_
    n, inf, nan = 700, float("inf"), float("nan")
    rows = [torch.ones(n), torch.zeros(n), torch.randn(n), torch.randn(n) * 1e-42, torch.randn(n), torch.arange(n).float()]
    rows[1][::2] = -0.0
    rows[2][5:400:3], rows[2][6:400:5] = inf, -inf
    rows[4][10:300:7], rows[4][300:500:3] = nan, -nan
    w = torch.stack(rows).to(DEV)[None]
    kc, vc, _ = _cache(1, n, len(rows), 64, torch.bfloat16, 0)
    lens = torch.tensor([n], device=DEV, dtype=torch.int32)
    kr, vr = kc.clone(), vc.clone()
    got = flash_attn_kvcache_evict_(kc, vc, lens, w, 257, sink=2, recent=31)
    want = ref.evict(kr, vr, lens, w, 257, 2, 31)
    assert torch.equal(got[2], want[2]) and torch.equal(kc, kr) and torch.equal(vc, vr)
    assert torch.equal(got[1].view(torch.int32), want[1].view(torch.int32))


def test_evict_leaves_lengths_outside_the_cache():
    from flash_attn import flash_attn_kvcache_evict_
    kc, vc, _ = _cache(3, 50, 2, 64, torch.bfloat16, 0)
    before = kc.clone()
    w = torch.rand(3, 2, 50, device=DEV)
    lens = torch.tensor([51, 50, -3], device=DEV, dtype=torch.int32)
    new, nw, kept = flash_attn_kvcache_evict_(kc, vc, lens, w, 20)
    assert new.tolist() == [51, 20, -3] and (kept[[0, 2]] == -1).all()
    assert torch.equal(kc[[0, 2]], before[[0, 2]]) and torch.equal(nw[[0, 2]], w[[0, 2]])


@pytest.mark.parametrize("page", [0, 5, 64])
@pytest.mark.parametrize("sq,hk,d", [(1, 2, 64), (13, 16, 64), (64, 8, 128), (200, 1, 256), (700, 2, 40)])
def test_commit(sq, hk, d, page):
    from flash_attn import flash_attn_kvcache_commit_
    b = 4
    lens = torch.tensor([0, 5, 100, 63], device=DEV, dtype=torch.int32)
    kc, vc, table = _cache(b, 100 + sq, hk, d, torch.bfloat16, page)
    slots = kc.shape[1] * (1 if table is None else table.shape[1])
    acc = torch.rand(b, sq, device=DEV) < 0.5
    acc[0], acc[1] = False, True
    w = torch.rand(b, hk, slots, device=DEV)
    kr, vr, wr = kc.clone(), vc.clone(), w.clone()
    new = flash_attn_kvcache_commit_(kc, vc, lens, acc, block_table=table, attn_weight=w)
    assert torch.equal(new, ref.commit(kr, vr, lens, acc, table, wr))
    assert torch.equal(kc, kr) and torch.equal(vc, vr) and torch.equal(w, wr)
    lens[2] = slots - sq + 1                  # no room: untouched
    kr = kc.clone()
    new = flash_attn_kvcache_commit_(kc, vc, lens, acc, block_table=table)
    assert int(new[2]) == int(lens[2]) and torch.equal(kc[2] if table is None else kc[table[2].long()],
                                                       kr[2] if table is None else kr[table[2].long()])


@pytest.mark.parametrize("page", [0, 16])
def test_serving_run(page):
    """Norm + rotary, tree attention with weights, commit and eviction after each other, as a server runs
    them: two sequences, five rounds, checked against the references at every step."""
    from flash_attn import flash_attn_kvcache_commit_, flash_attn_kvcache_evict_, flash_attn_kvcache_func
    from flash_attn.layers.qk_norm import QKNormRotary
    b, h, hk, d, sq, dtype = 2, 8, 2, 64, 9, torch.bfloat16
    torch.manual_seed(0)
    norm = QKNormRotary(d, d, device=DEV, dtype=dtype)
    kc, vc, table = _cache(b, 160, hk, d, dtype, page)
    slots = kc.shape[1] * (1 if table is None else table.shape[1])
    lens = torch.tensor([100, 37], device=DEV, dtype=torch.int32)
    place = lens.clone()                      # true positions: eviction does not change them
    w = torch.zeros(b, hk, slots, device=DEV)
    for step in range(5):
        qkv = torch.randn(b, sq, h + 2 * hk, d, device=DEV, dtype=dtype)
        mask = _tree(b, sq, step)
        depth = mask.sum(2).to(torch.int32) - 1
        with torch.no_grad():
            q, k = norm(qkv[:, :, :h], qkv[:, :, h:h + hk], place[:, None] + depth, max_position=1000)
            v = qkv[:, :, h + hk:]
            kr, vr, wr = kc.clone(), vc.clone(), w.clone()
            out, lse = flash_attn_kvcache_func(q, kc, vc, lens, k, v, block_table=table, tree_mask=mask, attn_weight=w,
                                               return_softmax_lse=True)
        r = ref.attention(q, kr, vr, lens, k, v, table, mask)
        _check(out, lse, None, r, dtype, d, 0, 0)
        torch.testing.assert_close(w.double(), wr.double() + r[2], rtol=1e-4, atol=1e-5)
        acc = mask[torch.arange(b), torch.randint(0, sq, (b,))]      # the path to some drafted token
        wr = w.clone()
        new = flash_attn_kvcache_commit_(kc, vc, lens, acc, block_table=table, attn_weight=w)
        assert torch.equal(new, ref.commit(kr, vr, lens, acc, table, wr)) and torch.equal(kc, kr) and torch.equal(w, wr)
        place += new - lens
        got = flash_attn_kvcache_evict_(kc, vc, new, w, 96, sink=4, recent=16, block_table=table)
        want = ref.evict(kr, vr, new, w, 96, 4, 16, table)
        assert all(torch.equal(a, x) for a, x in zip(got, want)) and torch.equal(kc, kr) and torch.equal(vc, vr)
        lens, w = got[0], got[1]


def test_graph_replays_two_graphs_and_streams():
    """Decode steps captured in two graphs over the same cache, replayed in turn with eager work between."""
    from flash_attn import flash_attn_kvcache_commit_, flash_attn_kvcache_evict_, flash_attn_kvcache_func
    b, h, hk, d = 2, 8, 2, 128
    torch.manual_seed(0)
    kc, vc, _ = _cache(b, 3000, hk, d, torch.bfloat16, 0)
    kept = kc.clone(), vc.clone()
    lens = torch.tensor([2500, 77], device=DEV, dtype=torch.int32)
    sizes = (1, 4)
    ins = [[torch.randn(b, s, n, d, device=DEV, dtype=torch.bfloat16) for n in (h, hk, hk)] for s in sizes]
    acc = [torch.ones(b, s, dtype=torch.bool, device=DEV) for s in sizes]

    def step(i, cache, lens):
        w = torch.zeros(b, hk, 3000, device=DEV)
        q, k, v = ins[i]
        out, lse = flash_attn_kvcache_func(q, *cache, lens, k, v, attn_weight=w, return_softmax_lse=True)
        new = flash_attn_kvcache_commit_(*cache, lens, acc[i], attn_weight=w)
        return [out, lse, new, *flash_attn_kvcache_evict_(*cache, new, w, 2000, sink=2, recent=5)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            step(i, (kc, vc), lens)
    torch.cuda.current_stream().wait_stream(side)
    graphs, held = [torch.cuda.CUDAGraph() for _ in sizes], []
    for i, g in enumerate(graphs):
        with torch.cuda.graph(g):
            held.append(step(i, (kc, vc), lens))
    for turn in range(4):
        i = turn % 2
        kc.copy_(kept[0]); vc.copy_(kept[1])
        lens.copy_(torch.tensor([2500 - 100 * turn, 77 + turn], dtype=torch.int32))
        ins[i][0].normal_()
        graphs[i].replay()
        torch.cuda.synchronize()
        cache = kept[0].clone(), kept[1].clone()
        want = step(i, cache, lens.clone())
        for a, x in zip(held[i], want):
            assert torch.equal(a, x)
        assert torch.equal(kc, cache[0]) and torch.equal(vc, cache[1])


def test_deterministic_and_split_independent_of_room():
    """Twice the same bits; a cache with more room may split the keys otherwise: fp32-close."""
    from flash_attn import flash_attn_kvcache_func
    torch.manual_seed(0)
    q = torch.randn(1, 4, 16, 128, device=DEV, dtype=torch.float16)
    base = torch.randn(2, 1, 60000, 2, 128, device=DEV, dtype=torch.float16)
    lens = torch.tensor([900], device=DEV, dtype=torch.int32)
    outs = [flash_attn_kvcache_func(q, base[0][:, :n], base[1][:, :n], lens, return_softmax_lse=True)
            for n in (60000, 60000, 904, 5000)]
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    for o in outs[2:]:
        torch.testing.assert_close(o[0].float(), outs[0][0].float(), atol=2.0 ** -11, rtol=2.0 ** -9)
        torch.testing.assert_close(o[1], outs[0][1], atol=2.0 ** -18, rtol=2.0 ** -18)


def test_misaligned_contiguous_rows():
    """q, k and v may start at any element: contiguous tensors off a 16-byte boundary give what aligned ones give."""
    from flash_attn import flash_attn_kvcache_func
    torch.manual_seed(0)
    q, k, v = (torch.randn(2, 3, h, 64, device=DEV, dtype=torch.float16) for h in (4, 2, 2))
    lens = torch.tensor([5, 33], device=DEV, dtype=torch.int32)

    def off(t):
        x = torch.empty(t.numel() + 3, device=DEV, dtype=t.dtype)[3:].view(t.shape)
        return x.copy_(t)

    caches = [torch.randn(2, 40, 2, 64, device=DEV, dtype=torch.float16) for _ in range(2)]
    outs = []
    for f in (lambda t: t, off):
        kc, vc = (c.clone() for c in caches)
        outs.append((flash_attn_kvcache_func(f(q), kc, vc, lens, k=f(k), v=f(v)), kc, vc))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_more_sequences_than_lanes():
    """The scan over the lengths goes past 64 sequences."""
    lens = [(37 * i) % 301 for i in range(150)]
    _run(150, 3, 4, 2, 64, lens, torch.bfloat16, 0)
    _run(150, 1, 2, 1, 128, lens, torch.float16, 32)


@pytest.mark.parametrize("page", [0, 24])
@pytest.mark.parametrize("d", [40, 128, 256])
def test_evict_many_heads(d, page):
    """As many heads as take the whole-line column slices of the move."""
    test_evict(16, d, [(97 * i) % 700 for i in range(16)], 150, 3, 20, page)
