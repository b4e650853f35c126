"""CPU checks of the key/value cache and norm + rotary entry points: what they refuse, and the cache
addressing the kernels share (csrc/fa_kvcache.h), compiled for the host."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from conftest import PKG


def _args(**over):
    bf = torch.bfloat16
    a = dict(q=torch.zeros(2, 3, 4, 64, dtype=bf), k_cache=torch.zeros(2, 50, 2, 64, dtype=bf),
             v_cache=torch.zeros(2, 50, 2, 64, dtype=bf), cache_seqlens=torch.zeros(2, dtype=torch.int32),
             k=torch.zeros(2, 3, 2, 64, dtype=bf), v=torch.zeros(2, 3, 2, 64, dtype=bf))
    a.update(over)
    return a


BF = torch.bfloat16
REFUSED = [
    (dict(k_cache=torch.zeros(2, 50, 2, 64), v_cache=torch.zeros(2, 50, 2, 64)), "only fp16 and bf16"),
    (dict(v_cache=torch.zeros(2, 50, 2, 64, dtype=torch.float16)), "same dtype"),
    (dict(v_cache=torch.zeros(2, 49, 2, 64, dtype=BF)), "must both be"),
    (dict(v_cache=torch.zeros(2, 2, 50, 64, dtype=BF).transpose(1, 2)), "same strides"),
    (dict(k_cache=torch.zeros(2, 50, 2, 60, dtype=BF), v_cache=torch.zeros(2, 50, 2, 60, dtype=BF)), "multiple of 8"),
    (dict(k_cache=torch.zeros(2, 50, 2, 264, dtype=BF), v_cache=torch.zeros(2, 50, 2, 264, dtype=BF)), "at most 256"),
    (dict(k_cache=torch.zeros(2, 50, 2, 68, dtype=BF)[..., :64], v_cache=torch.zeros(2, 50, 2, 68, dtype=BF)[..., :64]),
     "16-byte aligned"),
    (dict(k_cache=torch.zeros(2, 0, 2, 64, dtype=BF), v_cache=torch.zeros(2, 0, 2, 64, dtype=BF)), "empty"),
    (dict(cache_seqlens=torch.zeros(2, dtype=torch.int64)), "int32 vector"),
    (dict(cache_seqlens=torch.zeros(3, dtype=torch.int32)), "same batch size"),
    (dict(block_table=torch.zeros(2, 4, dtype=torch.int64)), "int32 \\(batch, blocks\\)"),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.int32)), "int32 \\(batch, blocks\\)"),
    (dict(block_table=torch.zeros(4, 2, dtype=torch.int32).t()), "contiguous last"),
    (dict(q=torch.zeros(2, 3, 4, 64, dtype=torch.float16)), "same dtype"),
    (dict(q=torch.zeros(2, 3, 3, 64, dtype=BF)), "must divide"),
    (dict(q=torch.zeros(2, 0, 4, 64, dtype=BF)), "at least one"),
    (dict(q=torch.zeros(2, 3, 4, 128, dtype=BF)), "q must have shape"),
    (dict(q=torch.zeros(2, 51, 4, 64, dtype=BF), k=None, v=None), "more drafted tokens"),
    (dict(k=None), "come together"),
    (dict(k=torch.zeros(2, 2, 2, 64, dtype=BF)), "k and v must have shape"),
    (dict(v=torch.zeros(2, 3, 2, 64, dtype=torch.float16)), "the cache's dtype"),
    (dict(tree_mask=torch.ones(3, 3)), "tree_mask must be bool"),
    (dict(tree_mask=torch.ones(3, 4, dtype=torch.bool)), "tree_mask must be bool"),
    (dict(attn_weight=torch.zeros(2, 3, 50)), "attn_weight must be fp32"),
    (dict(attn_weight=torch.zeros(2, 2, 2)), "more drafted tokens"),
    (dict(attn_weight=torch.zeros(2, 2, 50, dtype=BF)), "attn_weight must be fp32"),
    (dict(softmax_scale=0.0), "positive and finite"),
    (dict(softmax_scale=-1.0), "positive and finite"),
    (dict(softmax_scale=float("nan")), "positive and finite"),
    (dict(q=torch.zeros(2, 3, 4, 64, dtype=BF, requires_grad=True)), "no backward"),
    (dict(k_cache=torch.zeros(1, 50, 2, 64, dtype=BF).expand(2, -1, -1, -1),
          v_cache=torch.zeros(1, 50, 2, 64, dtype=BF).expand(2, -1, -1, -1)), "not be expanded"),
    (dict(attn_weight=torch.zeros(2, 1, 50).expand(-1, 2, -1)), "not be expanded"),
    (dict(attn_weight=torch.zeros(2, 2, 50, requires_grad=True)), "no backward"),
    (dict(), "on the GPU"),
]


@pytest.mark.parametrize("over,message", REFUSED, ids=[m for _, m in REFUSED])
def test_attention_refuses(over, message):
    from flash_attn import flash_attn_kvcache_func
    with pytest.raises(RuntimeError, match=message):
        flash_attn_kvcache_func(**_args(**over))


def test_shared_memory_is_refused():
    from flash_attn import flash_attn_kvcache_commit_, flash_attn_kvcache_evict_, flash_attn_kvcache_func
    from flash_attn.layers.qk_norm import apply_qk_norm_rotary_func
    a = _args()
    a["v_cache"] = a["k_cache"]
    with pytest.raises(RuntimeError, match="share memory"):
        flash_attn_kvcache_func(**a)
    with pytest.raises(RuntimeError, match="share memory"):
        flash_attn_kvcache_commit_(a["k_cache"], a["k_cache"].view_as(a["k_cache"]), a["cache_seqlens"],
                                   torch.ones(2, 3, dtype=torch.bool))
    one = torch.zeros(1, 50, 2, 64, dtype=BF).expand(2, -1, -1, -1)
    with pytest.raises(RuntimeError, match="not be expanded"):
        flash_attn_kvcache_evict_(one, one[:1].clone().expand(2, -1, -1, -1), a["cache_seqlens"], torch.zeros(2, 2, 50), 10)
    a["k"] = a["v"] = None                         # nothing is written: read all the same
    with pytest.raises(RuntimeError, match="on the GPU"):
        flash_attn_kvcache_func(**a)
    with pytest.raises(RuntimeError, match="share memory"):
        apply_qk_norm_rotary_func(a["q"], a["q"], inplace=True)
    with pytest.raises(RuntimeError, match="not be expanded"):
        apply_qk_norm_rotary_func(a["q"][:, :, :1].expand(-1, -1, 4, -1), a["q"], inplace=True)
    kv = torch.zeros(2, 3, 2, 4, 64, dtype=BF)     # halves of one tensor do not overlap
    with pytest.raises(RuntimeError, match="on the GPU"):
        apply_qk_norm_rotary_func(kv[:, :, 0], kv[:, :, 1], inplace=True)


def test_commit_and_evict_refuse():
    from flash_attn import flash_attn_kvcache_commit_, flash_attn_kvcache_evict_
    a = _args()
    cache = (a["k_cache"], a["v_cache"], a["cache_seqlens"])
    w = torch.zeros(2, 2, 50)
    for acc, message in ((torch.ones(2, 3), "accepted must be bool"), (torch.ones(3, 3, dtype=torch.bool), "batch"),
                         (torch.ones(2, 0, dtype=torch.bool), "between 1"), (torch.ones(2, 51, dtype=torch.bool), "between 1"),
                         (torch.ones(2, 3, dtype=torch.bool), "on the GPU")):
        with pytest.raises(RuntimeError, match=message):
            flash_attn_kvcache_commit_(*cache, acc)
    for kw, message in ((dict(budget=0), "budget"), (dict(budget=4, sink=3, recent=2), "budget"),
                        (dict(budget=4, sink=-1), "budget"), (dict(budget=4), "on the GPU")):
        with pytest.raises(RuntimeError, match=message):
            flash_attn_kvcache_evict_(*cache, w, **kw)
    with pytest.raises(RuntimeError, match="attn_weight"):
        flash_attn_kvcache_evict_(*cache, w[:, :1], 4)


def test_norm_rotary_refuses():
    from flash_attn.layers.qk_norm import apply_qk_norm_rotary_func as f
    q, k = torch.zeros(2, 5, 4, 64, dtype=BF), torch.zeros(2, 5, 2, 64, dtype=BF)
    w, cos = torch.ones(64), torch.ones(5, 32)
    pos = torch.zeros(2, 5, dtype=torch.int32)
    bad = [
        ((q.float(), k.float()), {}, "only fp16"), ((q, k.half()), {}, "same dtype"), ((q, k[0]), {}, "q and k must be"),
        ((q, k[:, :4]), {}, "agree"), ((q, k[..., :32]), {}, "agree"), ((q, k[:, :, :0]), {}, "a head each"),
        ((torch.zeros(1, 1, 1, 260, dtype=BF),) * 2, {}, "at most 256"), ((q.transpose(2, 3), k.transpose(2, 3)), {}, "agree|contig"),
        ((q, k, w[:32]), {}, "shape \\(headdim"), ((q, k, w.double()), {}, "fp32 or of q"),
        ((q, k, w, w.to(BF)), {}, "share a dtype"), ((q, k, w, w, cos), {}, "come together"),
        ((q, k, w, w, cos, cos[:, :16]), {}, "bad cos"), ((q, k, w, w, torch.ones(5, 33), torch.ones(5, 33)), {}, "bad cos"),
        ((q, k, w, w, cos.double(), cos.double()), {}, "fp32 or of q"), ((q, k, w, w, cos[:4], cos[:4]), {}, "fewer rows"),
        ((q, k, w, w, cos, cos, pos.long()), {}, "int32"), ((q, k, w, w, cos, cos, pos[:1]), {}, "shape of q"),
        ((q, k, w, w, None, None, pos), {}, "without cos"), ((q, k), dict(eps=-1.0), "negative"),
        ((q, k), dict(eps=float("nan")), "negative"), ((q, k, w, w, cos, cos, pos), {}, "on the GPU")]
    for args, kw, message in bad:
        with pytest.raises(RuntimeError, match=message):
            f(*args, **kw)


def test_c_abi_refuses_without_touching_memory():
    """Sizes outside the contract come back as false with a message (on a GPU box the device check passes
    and the sizes are refused; here the device is), and the workspace query as 0."""
    import flash_attn_2_cuda as m
    lib = m._lib
    P, I, L, F, B = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_bool
    z = (L * 3)(0, 0, 0)
    for name, kinds, args in (
            ("flash_attn_kvcache", [P] * 12 + [I] * 8 + [F] + [P] * 5 + [L] + [P] * 2 + [B, P],
             [None] * 12 + [1, 1, 1, 1, 1, 60, 0, 0, 1.0, z, z, z, z, z, 0, z, z, True, None]),
            ("flash_attn_kvcache_evict", [P] * 9 + [I] * 9 + [P, L, P, P, P],
             [None] * 9 + [1, 1, 1, 8, 0, 0, 0, 0, 0, z, 0, z, z, None]),
            ("flash_attn_kvcache_commit", [P] * 7 + [I] * 7 + [P, L, L, P, P],
             [None] * 7 + [1, 1, 1, 1, 8, 0, 0, z, 0, 0, z, None])):
        f = getattr(lib, name)
        f.argtypes, f.restype = kinds, B
        assert f(*args) is False, name
        assert lib.flash_attn_error()
    w = lib.flash_attn_kvcache_workspace
    w.argtypes, w.restype = [I] * 6 + [B], ctypes.c_size_t
    assert w(1, 1, 0, 1, 1, 64, False) == 0
    assert w(1, 1, 100, 3, 2, 64, False) == 0
    # small caches are never cut and need no workspace; long ones hold fp32 rows and their LSE
    assert w(1, 1, 100, 2, 2, 64, False) == 0
    size = w(1, 2, 65536, 4, 2, 128, False)
    assert size > 0 and size % (2 * 4 * 129 * 4) == 0
    assert w(1, 2, 65536, 4, 2, 128, True) == size + 2 * 4 * 65536 * 4


HOST = r"""
#include "fa_kvcache.h"
#include <cstdio>
#include <cstdlib>
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
  // every key of every sequence lands inside the cache, whatever the table and the lengths say
  const int b = 3, pages = 7, page = 5, blocks = 4, hk = 2, d = 64;
  int table[b * blocks] = {0, 6, 3, 1,  7, -1, 2147483647, -2147483647 - 1,  2, 4, 5, 7};
  fa::KvCache c{};
  c.table = table; c.table_row = blocks; c.page = page; c.num_pages = pages; c.slots = blocks * page;
  c.b = b; c.hk = hk; c.d = d; c.head = d; c.row = hk * d; c.batch = (int64_t)page * hk * d;
  const int64_t total = (int64_t)pages * page * hk * d;
  for (int s = 0; s < b; ++s)
    for (int j = 0; j < c.slots; ++j) {
      bool bad = false;
      const int64_t off = fa::slot_offset(c, s, j, bad);
      const int pg = table[s * blocks + j / page];
      CHECK(bad == (pg < 0 || pg >= pages));
      CHECK(off >= 0 && off + (hk - 1) * d + d <= total);
      if (!bad) CHECK(off == ((int64_t)pg * page + j % page) * hk * d);
    }
  // offsets past 32 bits
  c.table = nullptr; c.slots = 1 << 30; c.batch = (int64_t)c.slots * c.row;
  bool bad = false;
  CHECK(fa::slot_offset(c, 2, c.slots - 1, bad) == 3 * c.batch - c.row && !bad);
  // lengths
  c.slots = 100;
  const int lens[] = {0, 99, 100, 101, -1, 2147483647, -2147483647 - 1};
  const bool one[] = {true, true, false, false, false, false, false};
  for (int i = 0; i < 7; ++i) CHECK(fa::seq_ok(c, lens[i], 1) == one[i]);
  CHECK(fa::seq_ok(c, 100, 0) && !fa::seq_ok(c, 101, 0) && fa::seq_ok(c, 0, 100) && !fa::seq_ok(c, 1, 100));
  std::puts("ok");
  return 0;
}
"""


def test_cache_addressing_on_the_host(tmp_path):
    hipcc = "/opt/rocm/bin/hipcc"
    if shutil.which(hipcc) is None:
        pytest.skip("no hipcc")
    src, exe = tmp_path / "host.cpp", tmp_path / "host"
    src.write_text(HOST)
    subprocess.run([hipcc, "-x", "hip", "--cuda-host-only", "-std=c++17", "-I", os.path.join(PKG, "csrc"), str(src), "-o",
                    str(exe)], check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
