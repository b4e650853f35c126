"""GPU test of a refused capture: a variable-length forward whose work list the device builds raises while its
stream is being captured, nothing of it is replayed, and the same call outside the capture still runs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
def test_varlen_capture_is_refused(d):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from flash_attn import flash_attn_varlen_qkvpacked_func
    torch.manual_seed(0)
    qkv = torch.randn(4793, 3, 8, d, device="cuda", dtype=torch.bfloat16)
    cu = torch.tensor([0, 700, 2200, 2233, 4281, 4793], device="cuda", dtype=torch.int32)
    eager = flash_attn_varlen_qkvpacked_func(qkv, cu, 2048, causal=True)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            flash_attn_varlen_qkvpacked_func(qkv, cu, 2048, causal=True)
    assert torch.equal(flash_attn_varlen_qkvpacked_func(qkv, cu, 2048, causal=True), eager)
