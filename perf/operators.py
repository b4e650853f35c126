"""What the serving and normalisation operators are measured on: their cases, inputs, plain forms and exact values.

Four operators: the per-head norm of queries and keys with the rotary embedding in the same pass
("norm_rotary"), attention of drafted tokens over a key/value cache ("tree_attention"), eviction
from that cache by accumulated attention weight ("evict") and the commit of the accepted drafted
tokens ("commit").  With ``own`` false ``run`` computes them with elementary torch operations in
32 bits or more, rounded once at the end; with ``own`` true it calls the framework."""
import os
import sys

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # one new token of each of 16 sequences at far positions, grouped heads: latency counts
        _norm("norm_rotary_decode", b=16, s=1, h=32, hk=8, d=128, rd=128, dtype="bf16", table="fp32",
              positions=True, interleaved=False, backward=False),
        # one long prompt with an odd number of tokens, adjacent pairs, part of the head rotated
        _norm("norm_rotary_prefill_odd", b=1, s=8191, h=12, hk=3, d=96, rd=48, dtype="fp16", table="fp16",
              positions=False, interleaved=True, backward=False),
        # a training step of a packed projection with 16 heads of 64: outputs and all gradients
        _norm("norm_rotary_train_d64", b=4, s=2048, h=16, hk=16, d=64, rd=32, dtype="bf16", table="bf16",
              positions=False, interleaved=False, backward=True),
        # the largest training step: 8k tokens of 4 sequences, grouped heads of 128
        _norm("norm_rotary_train_large", b=4, s=8192, h=32, hk=8, d=128, rd=128, dtype="bf16", table="fp32",
              positions=False, interleaved=False, backward=True),
        # plain decoding of one sequence: one row over 4k keys
        _tree("decode_one", b=1, sq=1, h=32, hk=8, d=128, most=4096, least=4096, dtype="bf16", page=0,
              weight=False),
        # plain decoding of 8 ragged long sequences, with the weights that eviction goes by
        _tree("decode_long_weight", b=8, sq=1, h=32, hk=8, d=128, most=32768, least=20000, dtype="fp16",
              page=0, weight=True),
        # a tree of 48 drafted tokens for 16 sequences of a paged cache
        _tree("tree_paged", b=16, sq=48, h=32, hk=8, d=128, most=8192, least=1, dtype="bf16", page=64,
              weight=False),
        # a small tree, ungrouped heads of 64, short sequences (one of them empty) on pages of an odd size
        _tree("tree_short_odd", b=3, sq=13, h=16, hk=16, d=64, most=1531, least=0, dtype="fp16", page=17,
              weight=True),
        # one sequence that outgrew its budget by half
        _evict("evict_one", b=1, hk=8, d=128, most=4224, least=4224, budget=2048, sink=4, recent=256,
               dtype="bf16", page=0),
        # 8 long ragged sequences of a paged cache
        _evict("evict_long_paged", b=8, hk=8, d=128, most=32768, least=9001, budget=8192, sink=16,
               recent=1024, dtype="fp16", page=64),
        # the accepted tokens of one small tree
        _commit("commit_one", b=1, sq=13, hk=16, d=64, most=1531, least=1000, dtype="fp16", page=0),
        # the accepted tokens of a large batch of trees on a paged cache
        _commit("commit_batch_paged", b=128, sq=64, hk=8, d=128, most=2048, least=1, dtype="bf16", page=16),
    ]


def _norm(name, **sizes):
    return {"name": name, "op": "norm_rotary", **sizes}


def _tree(name, **sizes):
    return {"name": name, "op": "tree_attention", **sizes}


def _evict(name, **sizes):
    return {"name": name, "op": "evict", **sizes}


def _commit(name, **sizes):
    return {"name": name, "op": "commit", **sizes}


def _log_int(rng, low, high):
    """A whole number from [low, high], its logarithm spread evenly."""
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm_rotary", "tree_attention", "tree_attention", "evict", "commit"])
    dtype = rng.choice(["bf16", "fp16"])
    d = rng.choice([64, 128, 128, 8 * rng.randint(4, 32)])
    hk = rng.randint(1, 16)
    group = rng.randint(1, 8)
    page = rng.choice([0, 16, 64, rng.randint(1, 300)])
    if op == "norm_rotary":
        backward = rng.random() < 0.5
        b = _log_int(rng, 1, 32)
        room = 150_000_000 // (b * hk * (group + 1) * d)
        return {"op": op, "b": b, "s": _log_int(rng, 1, max(1, min(16384, room))), "h": hk * group, "hk": hk,
                "d": d, "rd": rng.choice([d, 2 * rng.randint(1, d // 2)]), "dtype": dtype,
                "table": rng.choice([dtype, "fp32"]), "positions": rng.random() < 0.5,
                "interleaved": rng.random() < 0.5, "backward": backward}
    b = _log_int(rng, 1, 32)
    room = max(64, 200_000_000 // (b * hk * d))
    if op == "tree_attention":
        sq = rng.choice([1, _log_int(rng, 1, 64)])
        room = max(64, min(room, 400_000_000_000 // (4 * b * hk * group * sq * d)))
        most = _log_int(rng, 16, min(65536, room))
        return {"op": op, "b": b, "sq": sq, "h": hk * group, "hk": hk, "d": d, "most": most,
                "least": rng.randint(0, most), "dtype": dtype, "page": page, "weight": rng.random() < 0.5}
    if op == "evict":
        most = _log_int(rng, 64, min(32768, room))
        budget = _log_int(rng, 16, most)
        sink = rng.randint(0, budget // 4)
        return {"op": op, "b": b, "hk": hk, "d": d, "most": most, "least": rng.randint(0, most),
                "budget": budget, "sink": sink, "recent": rng.randint(0, (budget - sink) // 2),
                "dtype": dtype, "page": page}
    most = _log_int(rng, 16, min(16384, room))
    return {"op": op, "b": b, "sq": _log_int(rng, 1, 128), "hk": hk, "d": d, "most": most,
            "least": rng.randint(0, most), "dtype": dtype, "page": page}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)


def _lengths(case, seed):
    """Cached keys of each sequence: the first has the most, the last the fewest."""
    r = np.random.RandomState(seed % (1 << 32))
    n = r.randint(case["least"], case["most"] + 1, case["b"])
    n[0], n[-1] = case["most"], case["least"] if case["b"] > 1 else case["most"]
    return torch.tensor(n, dtype=torch.int32, device=DEVICE)


def _cache(case, g, slots):
    """K and V caches with room for ``slots`` keys of each sequence, and the table of the pages."""
    b, page, dtype = case["b"], case["page"], TYPES[case["dtype"]]
    if page:
        blocks = -(-slots // page)
        shape = (b * blocks + 3, page, case["hk"], case["d"])
        table = torch.randperm(b * blocks + 3, generator=g, device=DEVICE)[:b * blocks]
        table = table.to(torch.int32).reshape(b, blocks)
    else:
        shape, table = (b, slots, case["hk"], case["d"]), None
    return _randn(g, shape, dtype), _randn(g, shape, dtype), table


def _tree_mask(b, sq, seed):
    """(b, sq, sq): token i sees itself and its ancestors in a random tree (a parent comes first)."""
    r = np.random.RandomState((seed + 1) % (1 << 32))
    m = np.zeros((b, sq, sq), dtype=bool)
    for i in range(sq):
        if i:
            m[:, i] = m[np.arange(b), r.randint(max(0, i - 4), i, b)]
        m[:, i, i] = True
    return torch.from_numpy(m).to(DEVICE)


def prepare(case, seed):
    g = _generator(seed)
    c, dtype = case, TYPES[case["dtype"]]
    st = {"case": case}
    if c["op"] == "norm_rotary":
        b, s, h, hk, d = c["b"], c["s"], c["h"], c["hk"], c["d"]
        # q and k as views of the packed projection; the gains of a trained norm are near one
        qkv = _randn(g, (b, s, h + 2 * hk, d), dtype) * 2
        st["q"], st["k"] = qkv[:, :, :h], qkv[:, :, h:h + hk]
        st["wq"] = (1 + 0.2 * _randn(g, (d,), torch.float32)).to(dtype)
        st["wk"] = (1 + 0.2 * _randn(g, (d,), torch.float32)).to(dtype)
        far = max(s, 131072) if c["positions"] else s
        inv = 10000.0 ** (-torch.arange(0, c["rd"], 2, device=DEVICE, dtype=torch.float64) / c["rd"])
        angle = torch.outer(torch.arange(far, device=DEVICE, dtype=torch.float64), inv)
        st["cos"], st["sin"] = angle.cos().to(TYPES[c["table"]]), angle.sin().to(TYPES[c["table"]])
        st["positions"] = None
        if c["positions"]:   # every sequence goes on from its own place
            start = torch.randint(0, far - s + 1, (b, 1), generator=g, device=DEVICE)
            st["positions"] = (start + torch.arange(s, device=DEVICE)).to(torch.int32)
        if c["backward"]:
            st["gq"], st["gk"] = _randn(g, (b, s, h, d), dtype), _randn(g, (b, s, hk, d), dtype)
        return st
    st["lens"] = _lengths(c, seed)
    if c["op"] == "tree_attention":
        b, sq, hk, d = c["b"], c["sq"], c["hk"], c["d"]
        slots = c["most"] + sq
        st["k_cache"], st["v_cache"], st["table"] = _cache(c, g, slots)
        st["q"] = _randn(g, (b, sq, c["h"], d), dtype)
        st["k"], st["v"] = _randn(g, (b, sq, hk, d), dtype), _randn(g, (b, sq, hk, d), dtype)
        st["mask"] = _tree_mask(b, sq, seed) if sq > 1 else None
        st["weight"] = None
        if c["weight"]:
            st["weight"] = torch.rand((b, hk, slots), generator=g, device=DEVICE)
    elif c["op"] == "evict":
        st["k_cache"], st["v_cache"], st["table"] = _cache(c, g, c["most"])
        # most of the weight lies on few keys, and some keys were never looked at
        w = torch.randn((c["b"], c["hk"], c["most"]), generator=g, device=DEVICE)
        st["weight"] = torch.where(w < -1.2, 0.0, torch.exp(2 * w))
    else:
        st["k_cache"], st["v_cache"], st["table"] = _cache(c, g, c["most"] + c["sq"])
        st["accepted"] = torch.rand((c["b"], c["sq"]), generator=g, device=DEVICE) < 0.4
    return st


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
_api = None


def _framework():
    global _api
    if _api is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xhy-flash-attention_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import flash_attn
        import flash_attn.layers.qk_norm
        _api = flash_attn
    return _api


def run(state):
    op = state["case"]["op"]
    if op == "norm_rotary":
        return _run_norm(state)
    if op == "tree_attention":
        return _run_tree(state)
    return _run_evict(state) if op == "evict" else _run_commit(state)


def _run_norm(st):
    c = st["case"]
    if own:
        f = _framework().layers.qk_norm.apply_qk_norm_rotary_func
        if not c["backward"]:
            return f(st["q"], st["k"], st["wq"], st["wk"], st["cos"], st["sin"], st["positions"],
                     c["interleaved"], EPS)
        leaves = [st[n].detach().requires_grad_() for n in ("q", "k", "wq", "wk")]
        out = f(*leaves, st["cos"], st["sin"], st["positions"], c["interleaved"], EPS)
        return tuple(out) + torch.autograd.grad(out, leaves, (st["gq"], st["gk"]))
    qo, qx, qr, qw = _norm_rotary(st["q"], st["wq"], st)
    ko, kx, kr, kw = _norm_rotary(st["k"], st["wk"], st)
    if not c["backward"]:
        return qo, ko
    dq, dwq = _norm_rotary_grad(st["gq"], qx, qr, qw, st)
    dk, dwk = _norm_rotary_grad(st["gk"], kx, kr, kw, st)
    return qo, ko, dq, dk, dwq, dwk


def _tables(st, s):
    """cos and sin in 32 bits of each row, with an axis for the heads."""
    if st["positions"] is None:
        return st["cos"][:s].float()[None, :, None], st["sin"][:s].float()[None, :, None]
    p = st["positions"].long()
    return st["cos"][p].float()[:, :, None], st["sin"][p].float()[:, :, None]


def _rotate(x, cos, sin, c):
    rd = c["rd"]
    if c["interleaved"]:
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, x[..., rd:]), -1)


def _norm_rotary(x, w, st):
    f, wf = x.float(), w.float()
    rstd = torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
    unit = f * rstd
    cos, sin = _tables(st, x.shape[1])
    return _rotate(unit * wf, cos, sin, st["case"]).to(x.dtype), unit, rstd, wf


def _norm_rotary_grad(g, unit, rstd, wf, st):
    cos, sin = _tables(st, g.shape[1])
    back = _rotate(g.float(), cos, -sin, st["case"])
    dw = (back * unit).sum((0, 1, 2), dtype=torch.float64)
    back = back * wf
    dx = rstd * (back - unit * (back * unit).mean(-1, keepdim=True))
    return dx.to(g.dtype), dw.to(g.dtype)


def _slots(st, index):
    """Rows of the flattened cache (all pages, or all sequences, one after another) of the keys index[b, ...]."""
    k, table = st["k_cache"], st["table"]
    batch = torch.arange(index.shape[0], device=index.device).reshape(-1, *[1] * (index.dim() - 1))
    if table is None:
        return batch * k.shape[1] + index
    return table.long()[batch, index // k.shape[1]] * k.shape[1] + index % k.shape[1]


def _run_tree(st):
    c = st["case"]
    if own:
        out, lse = _framework().flash_attn_kvcache_func(
            st["q"], st["k_cache"], st["v_cache"], st["lens"], k=st["k"], v=st["v"], block_table=st["table"],
            tree_mask=st["mask"], attn_weight=st["weight"], return_softmax_lse=True)
    else:
        out, lse = _tree_attention(st)
    return (out, lse, st["k_cache"], st["v_cache"]) + (() if st["weight"] is None else (st["weight"],))


def _tree_attention(st):
    c, q = st["case"], st["q"]
    b, sq, hk, d = c["b"], c["sq"], c["hk"], c["d"]
    group, most = c["h"] // hk, c["most"] + sq
    lens = st["lens"].long()
    fresh = _slots(st, lens[:, None] + torch.arange(sq, device=q.device))
    flat_k, flat_v = st["k_cache"].view(-1, hk, d), st["v_cache"].view(-1, hk, d)
    flat_k[fresh], flat_v[fresh] = st["k"], st["v"]
    at = torch.arange(most, device=q.device)
    index = at.expand(b, -1)
    if st["table"] is None:
        keys, values = st["k_cache"], st["v_cache"]
    else:
        rows = _slots(st, index)
        keys, values = flat_k[rows], flat_v[rows]
    there = at < lens[:, None] + sq
    keys = keys.float().transpose(1, 2)
    values = torch.where(there[:, :, None, None], values.float(), 0.0).transpose(1, 2)
    rows = q.float().view(b, sq, hk, group, d).permute(0, 2, 3, 1, 4).reshape(b, hk, group * sq, d)
    score = (torch.matmul(rows, keys.transpose(2, 3)) * d ** -0.5).view(b, hk, group, sq, most)
    j = at - lens[:, None]                       # place among the drafted tokens
    if st["mask"] is None:
        see = (j[:, None] <= torch.arange(sq, device=q.device)[:, None])
    else:
        drafted = torch.gather(st["mask"], 2, j.clamp(0, sq - 1)[:, None].expand(b, sq, most))
        see = (j[:, None] < 0) | (drafted & there[:, None])
    score = torch.where(see[:, None, None], score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    p = p / total
    lse = (top + torch.log(total)).squeeze(-1).reshape(b, c["h"], sq)
    out = torch.matmul(p.view(b, hk, group * sq, most), values).view(b, c["h"], sq, d)
    if st["weight"] is not None:
        st["weight"] += p.sum((2, 3))
    return out.transpose(1, 2).to(q.dtype).contiguous(), lse


def _run_evict(st):
    c = st["case"]
    if own:
        lens, weight, kept = _framework().flash_attn_kvcache_evict_(
            st["k_cache"], st["v_cache"], st["lens"], st["weight"], c["budget"], sink=c["sink"],
            recent=c["recent"], block_table=st["table"])
        return lens, weight, kept, st["k_cache"], st["v_cache"]
    lens, hk, budget = st["lens"].long(), c["hk"], c["budget"]
    at = torch.arange(c["most"], device=DEVICE)
    n = lens[:, None, None]
    held = (at < c["sink"]) | (at >= n - c["recent"])
    key = torch.where(held, float("inf"), st["weight"])
    key = torch.where(at < n, key, float("-inf"))
    kept = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    left = lens.clamp(max=budget)
    place = torch.arange(budget, device=DEVICE)
    used = (place < left[:, None])[:, None].expand(-1, hk, -1)
    kept = torch.sort(torch.where(used, kept, c["most"]), dim=-1).values   # in the cache's order
    kept = torch.where(used, kept, -1)
    weight = torch.zeros_like(st["weight"])
    weight[..., :budget] = torch.where(used, torch.gather(st["weight"], 2, kept.clamp(min=0)), 0.0)
    heads = torch.arange(hk, device=DEVICE)[None, :, None].expand(kept.shape)[used]
    source = _slots(st, kept.clamp(min=0))[used]
    target = _slots(st, place.expand(kept.shape))[used]
    for name in ("k_cache", "v_cache"):
        flat = st[name].view(-1, hk, c["d"])
        flat[target, heads] = flat[source, heads]
    return left.to(torch.int32), weight, kept.to(torch.int32), st["k_cache"], st["v_cache"]


def _run_commit(st):
    c = st["case"]
    if own:
        lens = _framework().flash_attn_kvcache_commit_(st["k_cache"], st["v_cache"], st["lens"], st["accepted"],
                                                       block_table=st["table"])
        return lens, st["k_cache"], st["v_cache"]
    lens, ok = st["lens"].long()[:, None], st["accepted"]
    count = ok.sum(1)
    source = _slots(st, lens + torch.arange(c["sq"], device=DEVICE))[ok]
    target = _slots(st, lens + (ok.long().cumsum(1) - 1).clamp(min=0))[ok]
    for name in ("k_cache", "v_cache"):
        flat = st[name].view(-1, c["hk"], c["d"])
        flat[target] = flat[source]
    return (st["lens"] + count).to(torch.int32), st["k_cache"], st["v_cache"]


# ------------------------------------------------------------------------------------------------
# work and exact values
# ------------------------------------------------------------------------------------------------
def _mean_length(c):
    return (c["most"] + c["least"]) / 2 if c["b"] > 1 else c["most"]


def work(case):
    c = case
    if c["op"] == "norm_rotary":
        rows, size = c["b"] * c["s"], 2 * c["d"] * (c["h"] + c["hk"])
        table = (rows if c["positions"] else c["s"]) * c["rd"] * (4 if c["table"] == "fp32" else 2)
        passes = 4 if c["backward"] else 2       # x, y; dy, dx
        return {"bytes": rows * size * passes + table, "flops": rows * size * passes * 2}
    keys = c["b"] * c["hk"] * _mean_length(c)
    if c["op"] == "tree_attention":
        new = c["b"] * c["sq"]
        data = (keys + 2 * new * c["hk"]) * 4 * c["d"] + new * c["h"] * (4 * c["d"] + 4)
        data += keys * 8 if c["weight"] else 0
        return {"bytes": data, "flops": 4 * c["sq"] * (c["h"] // c["hk"]) * c["d"] * (keys + new * c["hk"] / 2)}
    if c["op"] == "evict":
        over = max(0, c["most"] - c["budget"]) / max(1, c["most"] - c["least"]) if c["b"] > 1 else 1
        sequences = max(1.0, c["b"] * min(1.0, over)) if c["most"] > c["budget"] else 0
        moved = sequences * c["hk"] * (c["budget"] - c["sink"])
        return {"bytes": keys * 4 + c["b"] * c["hk"] * (4 * c["most"] + 4 * c["budget"]) + moved * 8 * c["d"],
                "flops": keys}
    rows = c["b"] * 0.4 * c["sq"] * c["hk"]
    return {"bytes": rows * 8 * c["d"] + c["b"] * c["sq"], "flops": rows}


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm_rotary": _exact_norm, "tree_attention": _exact_tree, "evict": _exact_evict,
            "commit": _exact_commit}[case["op"]](case, st)


def _exact_norm(c, st):
    # the rotation as a product of complex numbers; the gradients by differentiation of the definition
    def forward(x, w):
        y = w * x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["d"] + EPS)
        rd = c["rd"]
        pairs = y[..., :rd].unflatten(-1, (rd // 2, 2) if c["interleaved"] else (2, rd // 2))
        if not c["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        rows = slice(0, c["s"]) if st["positions"] is None else st["positions"].long()
        turn = torch.complex(st["cos"][rows].double(), st["sin"][rows].double()).unsqueeze(-2)
        z = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
        z = z if c["interleaved"] else z.transpose(-1, -2)
        return torch.cat((z.flatten(-2), y[..., rd:]), -1)

    leaves = [st[n].double().requires_grad_(c["backward"]) for n in ("q", "k", "wq", "wk")]
    out = (forward(leaves[0], leaves[2]), forward(leaves[1], leaves[3]))
    if not c["backward"]:
        return out
    return tuple(x.detach() for x in out) + torch.autograd.grad(out, leaves, (st["gq"].double(), st["gk"].double()))


def _row(st, b, j):
    """The cache's first two indices of key j of sequence b."""
    if st["table"] is None:
        return b, j
    page = st["k_cache"].shape[1]
    return st["table"][b].long()[j // page], j % page


def _exact_tree(c, st):
    b, sq, h, d = c["b"], c["sq"], c["h"], c["d"]
    group = h // c["hk"]
    out = torch.zeros(b, sq, h, d, dtype=torch.float64, device=DEVICE)
    lse = torch.zeros(b, h, sq, dtype=torch.float64, device=DEVICE)
    weight = None if st["weight"] is None else st["weight"].double()
    for i, n in enumerate(st["lens"].tolist()):
        at = _row(st, i, torch.arange(n, n + sq, device=DEVICE))
        st["k_cache"][at], st["v_cache"][at] = st["k"][i], st["v"][i]
        at = _row(st, i, torch.arange(n + sq, device=DEVICE))
        mask = torch.ones(sq, sq, dtype=torch.bool, device=DEVICE).tril() if st["mask"] is None else st["mask"][i]
        hidden = torch.cat((torch.zeros(sq, n, dtype=torch.bool, device=DEVICE), ~mask), 1)
        keys, values = st["k_cache"][at].double(), st["v_cache"][at].double()
        for head in range(h):
            s = st["q"][i, :, head].double() @ keys[:, head // group].T / d ** 0.5
            s = s.masked_fill(hidden, float("-inf"))
            lse[i, head] = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[i, head][:, None])
            out[i, :, head] = p @ values[:, head // group]
            if weight is not None:
                weight[i, head // group, :n + sq] += p.sum(0)
    return (out, lse, st["k_cache"], st["v_cache"]) + (() if weight is None else (weight,))


def _exact_evict(c, st):
    budget, hk = c["budget"], c["hk"]
    weight = torch.zeros_like(st["weight"])
    kept = torch.full((c["b"], hk, budget), -1, dtype=torch.int32, device=DEVICE)
    lens = st["lens"].tolist()
    host = st["weight"].double().cpu().numpy()
    for i, n in enumerate(lens):
        for head in range(hk):
            index = np.arange(n)
            if n > budget:
                middle = index[c["sink"]:n - c["recent"]]
                best = np.lexsort((middle, -host[i, head, middle]))[:budget - c["sink"] - c["recent"]]
                index = np.sort(np.concatenate((index[:c["sink"]], middle[best], index[n - c["recent"]:])))
            index = torch.from_numpy(index).to(DEVICE)
            m = index.numel()
            kept[i, head, :m] = index.to(torch.int32)
            weight[i, head, :m] = st["weight"][i, head, index]
            source, target = _row(st, i, index), _row(st, i, torch.arange(m, device=DEVICE))
            for name in ("k_cache", "v_cache"):
                cache = st[name][:, :, head]
                cache[target] = cache[source]
    left = torch.tensor([min(n, budget) for n in lens], dtype=torch.int32, device=DEVICE)
    return left, weight, kept, st["k_cache"], st["v_cache"]


def _exact_commit(c, st):
    lens = st["lens"].tolist()
    for i, n in enumerate(lens):
        taken = st["accepted"][i].nonzero().flatten()
        source, target = _row(st, i, n + taken), _row(st, i, n + torch.arange(taken.numel(), device=DEVICE))
        for name in ("k_cache", "v_cache"):
            st[name][target] = st[name][source]
    left = st["lens"] + st["accepted"].sum(1).to(torch.int32)
    return left, st["k_cache"], st["v_cache"]
