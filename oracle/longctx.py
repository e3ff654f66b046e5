"""Plain 64-bit restatements of the operators for long contexts: attention with a window and sinks, attention of drafted tokens
over a cache of pages, and the cache's bookkeeping.  Test infrastructure only."""
import math

import torch


def sink_mask(sq, sk, window, sinks, device='cpu'):
    """(queries, keys): the query stands at its index + keys - queries."""
    p = torch.arange(sq, device=device)[:, None] + (sk - sq)
    c = torch.arange(sk, device=device)[None]
    return (c <= p) & ((c > p - window) | (c < sinks))


def _softmax(x, seen):
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True) if x.shape[-1] else torch.full((*x.shape[:-1], 1), -math.inf, dtype=x.dtype, device=x.device)
    e = torch.where(seen, torch.exp(x - torch.where(top == -math.inf, 0.0, top)), 0.0)
    l = e.sum(-1, keepdim=True)
    lse = torch.where(l > 0, top + torch.log(l), math.inf)[..., 0]
    return torch.where(l > 0, e / torch.where(l > 0, l, 1.0), 0.0), lse


def attention(q, k, v, seen, scale):
    """q (Hq, n, D), k, v (Hk, m, D), seen (n, m): out, logsumexp, and the probabilities."""
    g = q.shape[0] // k.shape[0]
    k, v = (t.double().repeat_interleave(g, 0) for t in (k, v))
    p, lse = _softmax(torch.matmul(q.double(), k.transpose(1, 2)) * scale, seen.expand(q.shape[0], -1, -1))
    return torch.matmul(p, v), lse, p


def attention_grads(q, k, v, dout, seen, scale):
    """dQ, dK, dV from the formula."""
    hk, g = k.shape[0], q.shape[0] // k.shape[0]
    o, _, p = attention(q, k, v, seen, scale)
    kx, vx = (t.double().repeat_interleave(g, 0) for t in (k, v))
    do = dout.double()
    ds = p * (torch.matmul(do, vx.transpose(1, 2)) - (do * o).sum(-1, keepdim=True))
    dq = scale * torch.matmul(ds, kx)
    dk = scale * torch.matmul(ds.transpose(1, 2), q.double())
    dv = torch.matmul(p.transpose(1, 2), do)
    return dq, dk.view(hk, g, *dk.shape[1:]).sum(1), dv.view(hk, g, *dv.shape[1:]).sum(1)


def chain(parents, t):
    """The token and its ancestors, or None where it is not there."""
    out = [t]
    while True:
        p = parents[out[-1]]
        if p == -1:
            return out
        if not 0 <= p < out[-1]:
            return None
        out.append(p)


def tree_mask(length, tokens, parents, window, sinks):
    """(tokens, length + tokens): what each drafted token sees of the slots."""
    seen = torch.zeros(tokens, max(length, 0) + tokens, dtype=torch.bool)
    if length < 0:
        return seen
    parents = list(range(-1, tokens - 1)) if parents is None else parents
    for t in range(tokens):
        up = chain(parents, t)
        if up is None:
            continue
        at = length + len(up) - 1
        near = lambda pos: not window or pos > at - window or pos < sinks
        for s in range(length):
            seen[t, s] = near(s)
        for i, j in enumerate(up):
            seen[t, length + j] = near(at - i)
    return seen


def rows_of(cache, table_row, n):
    """The first n slots of a sequence as (heads, n, columns), zeros and False where there is no page."""
    pages, heads, slots, d = cache.shape
    out = torch.zeros(heads, n, d, dtype=cache.dtype)
    there = torch.zeros(n, dtype=torch.bool)
    for s in range(n):
        col = s // slots
        if col < len(table_row) and 0 <= table_row[col] < pages:
            out[:, s] = cache[table_row[col], :, s % slots]
            there[s] = True
    return out, there


def tree_attention(q, k_cache, v_cache, table, lengths, parents, window, sinks, scale):
    """Everything on the CPU; (sequences, Hq, tokens, D) out and (sequences, Hq, tokens) logsumexp, and sums of |P| |V|."""
    b, hq, t, _ = q.shape
    out = torch.zeros(b, hq, t, v_cache.shape[3], dtype=torch.float64)
    lse = torch.full((b, hq, t), math.inf, dtype=torch.float64)
    size = torch.zeros_like(out)
    for z in range(b):
        n = int(lengths[z])
        seen = tree_mask(n, t, None if parents is None else parents[z].tolist(), window, sinks)
        row = table[z].tolist()
        room = min(seen.shape[1], len(row) * k_cache.shape[2])
        seen = seen[:, :room]
        k, there = rows_of(k_cache, row, room)
        v, _ = rows_of(v_cache, row, room)
        seen = seen & there
        hidden = ~seen.any(0)
        k[:, hidden] = 0                       # what nobody sees may be anything
        v[:, hidden] = 0
        out[z], lse[z], p = attention(q[z], k, v, seen, scale)
        size[z] = torch.matmul(p, v.double().abs().repeat_interleave(hq // k.shape[0], 0))
    return out, lse, size
