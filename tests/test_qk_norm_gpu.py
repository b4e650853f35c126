"""GPU tests of the per-head norm with rotary embedding (csrc/fa_qknorm.hip) against the definition in
fp64.  Tolerances: the output's one rounding is half a step, eps / 2 |y| (fp16 below its normal range:
2^-25); the fp32 arithmetic in front of it is a chain of at most 256 + 20 roundings of the row's sum
of squares, halved by the square root, plus 8 more, each 2^-24 of the largest term: 2^-16 of it."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
CASES = [  # (b, s, h, hk, d, rotary_dim)
    (1, 1, 1, 1, 8, 8), (2, 1, 32, 8, 128, 128), (1, 257, 3, 1, 64, 32), (3, 17, 5, 5, 96, 48), (2, 33, 6, 2, 256, 64),
    (1, 40, 4, 2, 128, 54), (2, 9, 3, 3, 40, 40), (1, 65, 2, 1, 59, 22), (2, 100, 9, 3, 32, 16), (1, 7, 2, 2, 255, 254),
    (2, 31, 4, 4, 80, 0), (1, 129, 7, 1, 192, 192), (1, 5, 1, 1, 1, 0), (4, 300, 8, 4, 128, 64)]


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import flash_attn_2_cuda  # noqa: F401


def _func():
    from flash_attn.layers.qk_norm import apply_qk_norm_rotary_func
    return apply_qk_norm_rotary_func


def _table(rows, rd, dtype):
    if rd == 0:
        return None, None
    inv = 10000.0 ** (-torch.arange(0, rd, 2, device=DEV, dtype=torch.float64) / rd)
    a = torch.outer(torch.arange(rows, device=DEV, dtype=torch.float64), inv)
    return a.cos().to(dtype), a.sin().to(dtype)


def _ref(x, w, cos, sin, pos, interleaved, eps):
    """(output, pair magnitude) of the definition; x (b, s, h, d) fp64 leaf."""
    z = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    z = z if w is None else z * w
    if cos is None:
        return z
    rd = 2 * cos.shape[1]
    rows = torch.arange(x.shape[1], device=x.device).expand(x.shape[:2]) if pos is None else pos.long()
    c, s = cos.double()[rows][:, :, None], sin.double()[rows][:, :, None]
    if interleaved:
        a, b = z[..., 0:rd:2], z[..., 1:rd:2]
        y = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = z[..., :rd // 2], z[..., rd // 2:rd]
        y = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((y, z[..., rd:]), -1)


def _near(got, want, scale, what, eps=None):
    """|got - want| <= eps / 2 |want| + 2^-16 scale (scale: the largest term of each row)."""
    eps = torch.finfo(got.dtype).eps if eps is None else eps
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    tol = eps / 2 * want.abs() + 2.0 ** -16 * scale + tiny
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (what, float((err - tol).max()), float((err / tol.clamp(min=1e-300)).max()))


def _make(b, s, h, hk, d, dtype, seed=0):
    torch.manual_seed(seed)
    qkv = torch.randn(b, s, h + 2 * hk, d, device=DEV, dtype=torch.float32).mul(2).to(dtype)
    return qkv[:, :, :h], qkv[:, :, h:h + hk]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients(case, interleaved, dtype):
    b, s, h, hk, d, rd = case
    q, k = _make(b, s, h, hk, d, dtype)
    wdtype = torch.float32 if d % 3 else dtype
    wq, wk = (1 + 0.3 * torch.randn(d, device=DEV)).to(wdtype), (1 + 0.3 * torch.randn(d, device=DEV)).to(wdtype)
    cos, sin = _table(s + 50, rd, torch.float32 if d % 16 else dtype)
    pos = None
    if s % 2 and rd:
        pos = torch.randint(0, s + 50, (b, s), device=DEV, dtype=torch.int32)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    out = _func()(*leaves, cos, sin, pos, interleaved, 1e-5)
    g = [torch.randn(b, s, n, d, device=DEV).to(dtype) for n in (h, hk)]
    grads = torch.autograd.grad(out, leaves, g)
    for i in range(2):
        x, w = leaves[i].detach().double().requires_grad_(), leaves[2 + i].detach().double().requires_grad_()
        y = _ref(x, w, cos, sin, pos, interleaved, 1e-5)
        gx, gw = torch.autograd.grad(y, (x, w), g[i].double())
        assert out[i].is_contiguous() and out[i].dtype == dtype
        _near(out[i], y.detach(), 2 * y.detach().abs().amax(-1, keepdim=True), "out")
        r = 1 / torch.sqrt(x.detach().square().mean(-1, keepdim=True) + 1e-5)
        top = g[i].double().abs().amax(-1, keepdim=True) * w.detach().abs().max()
        n = (x.detach() * r).abs().amax(-1, keepdim=True)
        _near(grads[i], gx, 4 * r * top * (1 + n), "dx")
        # fp32 sums of b s heads rows: at most 2^12 of them one after another here
        mass = (2 * g[i].double().abs().amax(-1, keepdim=True) * (x.detach() * r).abs()).sum((0, 1, 2))
        assert grads[2 + i].dtype == wdtype
        _near(grads[2 + i], gw, mass * 2.0 ** 4, "dw")


def test_gradient_against_differences():
    """dx and dw of a smooth function of the outputs against central differences of the fp64 formula."""
    q, k = _make(1, 3, 2, 1, 64, torch.float16)
    w = torch.linspace(0.5, 1.5, 64, device=DEV)
    cos, sin = _table(3, 32, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (q, k)] + [w.clone().requires_grad_(), w.clone().requires_grad_()]
    out = _func()(*leaves, cos, sin)
    c = [torch.randn_like(o) for o in out]
    grads = torch.autograd.grad(out, leaves, c)

    def f(i, x, ww):
        return float((_ref(x, ww, cos, sin, None, False, 1e-6) * c[i].double()).sum())

    for i in range(2):
        x, ww = leaves[i].detach().double(), w.double()
        for _ in range(8):
            dx, dwv = torch.randn_like(x), torch.randn_like(ww)
            e = 1e-6
            nx = (f(i, x + e * dx, ww) - f(i, x - e * dx, ww)) / (2 * e)
            nw = (f(i, x, ww + e * dwv) - f(i, x, ww - e * dwv)) / (2 * e)
            # each of the n rounded gradients is off by at most half a step (2^-11) of itself
            tx = float((grads[i].double() * dx).abs().sum()) * 2.0 ** -10 + 1e-4
            tw = float((grads[2 + i].double() * dwv).abs().sum()) * 2.0 ** -16 + 1e-4
            assert abs(float((grads[i].double() * dx).sum()) - nx) <= tx
            assert abs(float((grads[2 + i].double() * dwv).sum()) - nw) <= tw


def test_gradients_of_some_inputs_and_twice():
    """Each subset of weights and leaves gives the full call's gradients; a second differentiation raises."""
    q, k = (t.contiguous() for t in _make(1, 12, 4, 2, 64, torch.bfloat16))
    w = [(1 + 0.2 * torch.randn(64, device=DEV)) for _ in range(2)]
    cos, sin = _table(12, 64, torch.float32)
    g = [torch.randn_like(q), torch.randn_like(k)]

    def run(need, weights):
        leaves = [t.clone().requires_grad_(n) for t, n in zip((q, k, *w), need)]
        ww = [leaves[2 + i] if weights[i] else None for i in range(2)]
        out = _func()(leaves[0], leaves[1], *ww, cos, sin)
        torch.autograd.backward(out, g)
        return [t.grad for t in leaves]

    full = run((True,) * 4, (True, True))
    for need in ((True, False, False, False), (False, False, False, True), (False, True, True, False)):
        for a, b, n in zip(run(need, (True, True)), full, need):
            assert (torch.equal(a, b) if n else a is None)
    only_k = run((False, False, False, True), (False, True))
    assert torch.equal(only_k[3], full[3]) and only_k[2] is None
    leaf = q.clone().requires_grad_()
    out = _func()(leaf, k, w[0], None, cos, sin)[0]
    grad, = torch.autograd.grad(out.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        grad.sum().backward()


@pytest.mark.parametrize("d,rd", [(128, 128), (40, 22)])
def test_forms_agree(d, rd):
    """No weights, one weight, no batch dimension, in place, positions 0 .. s-1: one result."""
    f = _func()
    q, k = _make(1, 19, 6, 2, d, torch.bfloat16)
    cos, sin = _table(19, rd, torch.float32)
    one = torch.ones(d, device=DEV)
    want = f(q, k, one, one, cos, sin)
    pos = torch.arange(19, device=DEV, dtype=torch.int32)
    for got in (f(q, k, None, None, cos, sin), f(q, k, one, None, cos, sin), f(q, k, None, one, cos, sin),
                f(q, k, one, one, cos, sin, pos[None])):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = f(q[0], k[0], one, one, cos, sin, pos)
    assert all(torch.equal(a, b[0]) for a, b in zip(got, want))
    qi, ki = q.clone(), k.clone()
    got = f(qi, ki, one, one, cos, sin, inplace=True)
    assert got[0] is qi and got[1] is ki and torch.equal(qi, want[0]) and torch.equal(ki, want[1])


def test_inplace_on_packed_leaves_the_rest():
    qkv = torch.randn(2, 5, 8, 64, device=DEV, dtype=torch.bfloat16)
    keep = qkv.clone()
    cos, sin = _table(5, 64, torch.float32)
    want = _func()(qkv[:, :, :4], qkv[:, :, 4:6], None, None, cos, sin)
    _func()(qkv[:, :, :4], qkv[:, :, 4:6], None, None, cos, sin, inplace=True)
    assert torch.equal(qkv[:, :, :4], want[0]) and torch.equal(qkv[:, :, 4:6], want[1])
    assert torch.equal(qkv[:, :, 6:], keep[:, :, 6:])


def test_unaligned_strides_and_expanded_gradient():
    base = torch.randn(2, 11, 5, 70, device=DEV, dtype=torch.float16)
    q, k = base[..., 3:67][:, :, :3], base[..., 3:67][:, :, 3:]
    cos, sin = _table(11, 64, torch.float16)
    got = _func()(q, k, None, None, cos, sin)
    want = _func()(q.contiguous(), k.contiguous(), None, None, cos, sin)
    for a, b in zip(got, want):   # the 64-lane and the 16-byte form sum a row in another order
        torch.testing.assert_close(a, b, rtol=2.0 ** -10, atol=2.0 ** -12)
    ql = q.contiguous().requires_grad_()
    out = _func()(ql, k, None, None, cos, sin)
    out[0].sum().backward()
    gx = torch.autograd.grad(_ref(x := ql.detach().double().requires_grad_(), None, cos, sin, None, False, 1e-6).sum(), x)[0]
    torch.testing.assert_close(ql.grad.double(), gx, rtol=2.0 ** -10, atol=1e-4)


def test_position_outside_the_table_is_nan_and_zero_rows():
    q, k = _make(1, 4, 2, 1, 64, torch.bfloat16)
    q, k = q.clone(), k.clone()
    q[0, 2] = 0
    cos, sin = _table(10, 64, torch.float32)
    pos = torch.tensor([[0, 10, 9, -1]], device=DEV, dtype=torch.int32)
    oq, ok = _func()(q, k, None, None, cos, sin, pos)
    assert torch.isnan(oq[0, [1, 3]]).all() and torch.isnan(ok[0, [1, 3]]).all()
    assert torch.isfinite(oq[0, [0, 2]]).all() and (oq[0, 2] == 0).all()


def test_no_rows():
    q, k = torch.empty(2, 0, 4, 64, device=DEV, dtype=torch.bfloat16), torch.empty(2, 0, 2, 64, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(64, device=DEV, requires_grad=True)
    oq, ok = _func()(q.requires_grad_(), k, w, None)
    assert oq.shape == q.shape
    oq.sum().backward()
    assert (w.grad == 0).all()


def test_graph_replays_and_streams():
    q, k = (t.contiguous() for t in _make(2, 64, 8, 2, 128, torch.bfloat16))
    w = (1 + 0.1 * torch.randn(128, device=DEV))
    cos, sin = _table(64, 128, torch.float32)
    f = _func()
    ql, kl, wl = q.clone().requires_grad_(), k.clone().requires_grad_(), w.clone().requires_grad_()
    gq, gk = torch.randn_like(q), torch.randn_like(k)

    def step():
        out = f(ql, kl, wl, None, cos, sin)
        return (*out, *torch.autograd.grad(out, (ql, kl, wl), (gq, gk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [t.detach().clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [t.detach() for t in step()]
    for i in range(3):
        with torch.no_grad():
            ql.copy_(q * (i + 1) + i)
        graph.replay()
        torch.cuda.synchronize()
        want = [t.detach() for t in step()]
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    with torch.no_grad():
        ql.copy_(q)
    assert all(torch.equal(a, b.detach()) for a, b in zip(other, step()))


def test_many_rows_deterministic():
    q, k = _make(4, 1031, 16, 4, 128, torch.bfloat16)
    w = torch.ones(128, device=DEV, requires_grad=True)
    runs = []
    for _ in range(2):
        out = _func()(q, k, w, w)
        runs.append(torch.autograd.grad(out, w, [torch.ones_like(o) for o in out])[0])
    assert torch.equal(*runs)


def test_module_and_refusals():
    from flash_attn.layers.qk_norm import QKNormRotary
    m = QKNormRotary(64, 32, device=DEV, dtype=torch.float32)
    q, k = _make(2, 9, 4, 2, 64, torch.float16)
    cos, sin = _table(9, 32, torch.float32)
    want = _func()(q, k, m.q_weight, m.k_weight, cos, sin)
    assert all(torch.equal(a, b) for a, b in zip(m(q, k), want))
    pos = torch.randint(0, 500, (2, 9), device=DEV, dtype=torch.int32)
    cos, sin = _table(500, 32, torch.float32)
    want = _func()(q, k, m.q_weight, m.k_weight, cos, sin, pos)
    assert all(torch.equal(a, b) for a, b in zip(m(q, k, pos, max_position=500), want))
    with pytest.raises(RuntimeError, match="backward needs"):
        _func()(q, k, m.q_weight, m.k_weight, inplace=True)
    with pytest.raises(RuntimeError, match="fewer rows"):
        _func()(q, k, None, None, cos[:8], sin[:8])


def test_capture_beside_an_eager_graph_is_refused():
    """The accumulators that an eager graph of the same leaves keeps alive belong to its stream, which a captured
    backward could not leave: the captured forward is refused, and taken once that graph is gone."""
    q, k = (t.contiguous() for t in _make(1, 9, 4, 2, 64, torch.bfloat16))
    cos, sin = _table(9, 64, torch.float32)
    w = torch.ones(64, device=DEV, requires_grad=True)
    eager = _func()(q, k, w, w, cos, sin)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
            _func()(q, k, w, w, cos, sin)
        with torch.no_grad():                      # nothing to differentiate: nothing to refuse
            _func()(q, k, w, w, cos, sin)
    want = [t.detach().clone() for t in eager]
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _func()(q, k, w, w, cos, sin)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
