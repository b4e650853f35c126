"""Forward-mode tangents: the operators have none, and a dual input is refused, not answered without a tangent
(on a box without a GPU: before the device is looked at)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from flash_attn import flash_attn_kvcache_commit_, flash_attn_kvcache_evict_, flash_attn_kvcache_func
from flash_attn.layers.qk_norm import apply_qk_norm_rotary_func

BF = torch.bfloat16


def _dual(t):
    return fwd.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("no_grad", [False, True])
def test_tangents_are_refused(no_grad):
    q, k = torch.zeros(2, 3, 4, 64, dtype=BF), torch.zeros(2, 3, 2, 64, dtype=BF)
    cache = torch.zeros(2, 50, 2, 64, dtype=BF), torch.zeros(2, 50, 2, 64, dtype=BF)
    lens, w = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, 50)
    gain, cos = torch.ones(64), torch.ones(5, 32)
    with fwd.dual_level(), torch.set_grad_enabled(not no_grad):
        for args in ((_dual(q), k), (q, _dual(k)), (q, k, _dual(gain)), (q, k, None, _dual(gain)),
                     (q, k, gain, gain, _dual(cos), cos), (q, k, gain, gain, cos, _dual(cos))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                apply_qk_norm_rotary_func(*args)
        with pytest.raises(RuntimeError, match="forward-mode"):
            apply_qk_norm_rotary_func(_dual(q), k, inplace=True)
        for args in ((_dual(q), *cache, lens, k, k), (q, _dual(cache[0]), cache[1], lens, k, k),
                     (q, *cache, lens, _dual(k), k), (q, *cache, lens, k, k, None, None, None, _dual(w))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                flash_attn_kvcache_func(*args)
        with pytest.raises(RuntimeError, match="forward-mode"):
            flash_attn_kvcache_commit_(cache[0], _dual(cache[1]), lens, torch.ones(2, 3, dtype=torch.bool))
        with pytest.raises(RuntimeError, match="forward-mode"):
            flash_attn_kvcache_evict_(*cache, lens, _dual(w), 10)
        with pytest.raises(RuntimeError, match="on the GPU"):   # no tangent: no refusal
            apply_qk_norm_rotary_func(q, k)
        with pytest.raises(RuntimeError, match="on the GPU"):
            flash_attn_kvcache_evict_(*cache, lens, w, 10)
