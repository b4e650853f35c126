"""The cos / sin table that QKNormRotary keeps, over the calls of a module's life."""
import pytest
import torch

from flash_attn.layers.qk_norm import QKNormRotary


def test_table_made_under_inference_mode_is_an_ordinary_tensor():
    m = QKNormRotary(64, 32)
    with torch.inference_mode():
        cos, sin = m.table(20, torch.device("cpu"))
    assert not cos.is_inference() and not sin.is_inference()
    again = m.table(20, torch.device("cpu"))
    assert again[0] is cos and again[1] is sin
    x = torch.randn(20, 16, requires_grad=True)
    (x * cos).sum().backward()                     # saved for a backward


@pytest.mark.gpu
def test_training_after_generation_under_inference_mode():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    m = QKNormRotary(64, 32, device="cuda")
    q, k = (torch.randn(2, 20, h, 64, device="cuda", dtype=torch.float16) for h in (4, 2))
    with torch.inference_mode():
        want = m(q, k)
    got = m(q, k)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    sum(t.float().sum() for t in got).backward()
    assert torch.isfinite(m.q_weight.grad).all() and (m.k_weight.grad != 0).any()


def test_outgrown_tables_stay():
    """A graph captured with a table reads it at every replay: its memory may not go to others."""
    import weakref
    m = QKNormRotary(64, 32)
    first = weakref.ref(m.table(20, torch.device("cpu"))[0])
    cos, sin = m.table(50, torch.device("cpu"))
    assert cos.shape[0] >= 50 and first() is not None
    assert torch.equal(first(), cos[:20]) and m.table(20, "cpu")[0] is cos


@pytest.mark.gpu
def test_captured_step_keeps_its_table():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    m = QKNormRotary(64, 64, device="cuda")
    q, k = (torch.randn(2, 20, h, 64, device="cuda", dtype=torch.float16) for h in (4, 2))
    pos = torch.randint(0, 64, (2, 20), device="cuda", dtype=torch.int32)
    with torch.no_grad():
        want = [t.clone() for t in m(q, k, pos, max_position=64)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(q, k, pos, max_position=64)
        for rows in (100, 5000):                   # longer calls on the same module
            m(q, k, pos, max_position=rows)
            over = [torch.full((64 * 32 + i,), float("nan"), device="cuda") for i in range(50)]
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            del over
        assert all(torch.equal(a, b) for a, b in zip(m(q, k, pos, max_position=64), want))


@pytest.mark.gpu
def test_table_that_a_capture_fills_serves_no_other_call():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    m = QKNormRotary(64, 64, device="cuda")
    q, k = (torch.randn(2, 20, h, 64, device="cuda", dtype=torch.float16) for h in (4, 2))
    pos = torch.randint(0, 64, (2, 20), device="cuda", dtype=torch.int32)
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(q, k, pos, max_position=64)
        want = [t.clone() for t in m(q, k, pos, max_position=64)]   # before the first replay
        cos = m.table(64, "cuda")[0]
        assert (cos[0] == 1).all() and cos.abs().max() <= 1
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            assert all(torch.equal(a, b) for a, b in zip(m(q, k, pos, max_position=64), want))


@pytest.mark.gpu
def test_table_made_on_a_busy_stream_serves_others_at_once():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    m = QKNormRotary(64, 64, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(int(2e8))                # the table's kernels wait behind this
        m.table(1000, "cuda")
    got = [t.clone() for t in m.table(1000, "cuda")]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, m.table(1000, "cuda")))
