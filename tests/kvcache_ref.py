"""fp64 references of the key/value cache operators, one sequence and head at a time, on any device."""
import torch


def slot(cache, table, b, j):
    """Index of the first two cache dims for key(s) j of sequence b."""
    if table is None:
        return b, j
    page = cache.shape[1]
    return table[b].long()[j // page], j % page


def attention(q, k_cache, v_cache, lens, k=None, v=None, table=None, mask=None, scale=None):
    """out, lse, weight (probability mass per key), bound terms.  The caches are changed as the call does.

    terms: sum_j p_j |v_j| and the largest sum |q k| scale of a row: what the tolerances count."""
    b, sq, h, d = q.shape
    hk = k_cache.shape[2]
    slots = k_cache.shape[1] * (1 if table is None else table.shape[1])
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(b, sq, h, d, dtype=torch.float64, device=q.device)
    lse = torch.full((b, h, sq), float("inf"), dtype=torch.float64, device=q.device)
    weight = torch.zeros(b, hk, slots, dtype=torch.float64, device=q.device)
    mass, score = torch.zeros_like(out), torch.zeros_like(lse)
    for i, n in enumerate(lens.tolist()):
        at = slot(k_cache, table, i, torch.arange(n, n + sq, device=q.device))
        if k is not None:
            k_cache[at], v_cache[at] = k[i], v[i]
        at = slot(k_cache, table, i, torch.arange(n + sq, device=q.device))
        see = torch.ones(sq, sq, dtype=torch.bool, device=q.device).tril() if mask is None else mask.expand(b, sq, sq)[i]
        see = torch.cat((torch.ones(sq, n, dtype=torch.bool, device=q.device), see), 1)
        seen = see.any(0)
        kk = torch.where(seen[:, None, None], k_cache[at].double(), 0.0)
        vv = torch.where(seen[:, None, None], v_cache[at].double(), 0.0)
        for head in range(h):
            kh = kk[:, head // (h // hk)]
            s = (q[i, :, head].double() @ kh.T * scale).masked_fill(~see, float("-inf"))
            some = see.any(1)
            p = torch.zeros_like(s)
            le = torch.logsumexp(s, 1)
            p[some] = torch.exp(s[some] - le[some][:, None])
            lse[i, head] = torch.where(some, le, float("inf"))
            vh = vv[:, head // (h // hk)]
            out[i, :, head] = p @ vh
            mass[i, :, head] = p @ vh.abs()
            score[i, head] = (q[i, :, head].double().abs() @ kh.abs().T * scale).amax(1)
            weight[i, head // (h // hk), :n + sq] += p.sum(0)
    return out, lse, weight, mass, score


def evict(k_cache, v_cache, lens, weight, budget, sink, recent, table=None):
    b, hk = weight.shape[:2]
    new, kept = weight.clone(), torch.full((b, hk, budget), -1, dtype=torch.int32, device=weight.device)
    left = lens.clone()
    for i, n in enumerate(lens.tolist()):
        new[i, :, n:] = 0
        left[i] = min(n, budget)
        for head in range(hk):
            idx = list(range(n))
            if n > budget:
                w = weight[i, head].double().cpu().tolist()
                key = {j: (0 if w[j] != w[j] else 1, 0.0 if w[j] != w[j] else -w[j], j) for j in idx}   # NaN first
                mid = sorted(idx[sink:n - recent], key=key.get)[:budget - sink - recent]
                idx = idx[:sink] + sorted(mid) + idx[n - recent:]
            t = torch.tensor(idx, device=weight.device, dtype=torch.long)
            m = len(idx)
            kept[i, head, :m] = t.to(torch.int32)
            new[i, head] = 0
            new[i, head, :m] = weight[i, head, t]
            src, dst = slot(k_cache, table, i, t), slot(k_cache, table, i, torch.arange(m, device=weight.device))
            for c in (k_cache, v_cache):
                c[:, :, head][dst] = c[:, :, head][src]
    return left, new, kept


def commit(k_cache, v_cache, lens, accepted, table=None, weight=None):
    for i, n in enumerate(lens.tolist()):
        t = accepted[i].nonzero().flatten()
        m = t.numel()
        src, dst = slot(k_cache, table, i, n + t), slot(k_cache, table, i, n + torch.arange(m, device=t.device))
        for c in (k_cache, v_cache):
            c[dst] = c[src]
        if weight is not None:
            w = weight[i, :, n + t].clone()
            weight[i, :, n:n + accepted.shape[1]] = 0
            weight[i, :, n:n + m] = w
    return lens + accepted.sum(1).to(lens.dtype)
