"""GPU test of a captured norm + rotary step beside accumulators that live on a side stream, as a data-parallel
wrapper made there holds them for life: the capture takes that stream in and lets it go again."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("into_grad", [False, True])
def test_capture_beside_accumulators_of_a_side_stream(into_grad):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from flash_attn.layers.qk_norm import apply_qk_norm_rotary_func as f
    q, k = (torch.randn(1, 9, h, 64, device="cuda", dtype=torch.bfloat16) for h in (4, 2))
    w = torch.ones(64, device="cuda", requires_grad=True)
    g = [torch.randn_like(t) for t in (q, k)]
    static = q.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held = f(static, k, w, w)                  # keeps w's accumulator, of this stream, alive
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f(static, k, w, w)
        if into_grad:
            torch.autograd.backward(out, g)
            grad = w.grad
        else:
            grad, = torch.autograd.grad(out, w, g)
    for i in range(3):
        static.copy_(q * (i + 1) + i)
        if into_grad:
            grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        leaf = w.detach().clone().requires_grad_()
        want = f(static, k, leaf, leaf)
        torch.autograd.backward(want, g)
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(grad, leaf.grad)
    del held
