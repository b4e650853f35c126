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
