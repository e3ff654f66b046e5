"""Plain 64-bit restatements of attention over keys and values from one latent vector a token, and of the bookkeeping of a batch's rows.
Test infrastructure only."""
import math

import torch

from . import longctx


def mask(sq, sk, causal, device='cpu'):
    """(queries, keys): the queries stand at the last keys."""
    if not causal:
        return torch.ones(sq, sk, dtype=torch.bool, device=device)
    return longctx.sink_mask(sq, sk, max(sq, sk) + 1, 0, device=device)


def keys(k, shared):
    """(heads, rows, E) and (rows, R) -> (heads, rows, E + R)"""
    return torch.cat([k, shared[None].expand(k.shape[0], -1, -1)], 2)


def attention(q, k, v, shared, causal, scale):
    """One sequence: out, logsumexp, probabilities."""
    return longctx.attention(q, keys(k, shared), v, mask(q.shape[1], k.shape[1], causal, q.device), scale)


def attention_grads(q, k, v, shared, dout, causal, scale):
    """dQ, dK, dV, and of the shared part of the keys, from the formula."""
    dq, dk, dv = longctx.attention_grads(q, keys(k, shared), v, dout, mask(q.shape[1], k.shape[1], causal, q.device), scale)
    e = k.shape[2]
    return dq, dk[..., :e], dv, dk[..., e:].sum(0)


def cache_attention(q, latent, table, lengths, starts, value_dim, scale):
    """(rows, Hq, E) over (pages, 1, slots, E), everything on the CPU: out, logsumexp, sums of |P| |value|."""
    rows, hq, _ = q.shape
    out = torch.zeros(rows, hq, value_dim, dtype=torch.float64)
    size = torch.zeros_like(out)
    lse = torch.full((rows, hq), math.inf, dtype=torch.float64)
    slots = latent.shape[2]
    for z, n in enumerate(lengths.tolist()):
        a, b = int(starts[z]), int(starts[z + 1])
        if n < 0 or a == b:
            continue
        room = min(n + b - a, table.shape[1] * slots)
        x, there = longctx.rows_of(latent, table[z].tolist(), room)
        x = torch.where(there[:, None], x[0].double(), 0.0)
        for t in range(b - a):
            seen = there & (torch.arange(room) <= n + t)
            o, l, p = longctx.attention(q[a + t][:, None], x[None], x[None, :, :value_dim], seen[None], scale)
            out[a + t], lse[a + t] = o[:, 0], l[:, 0]
            size[a + t] = torch.matmul(p, x[None, :, :value_dim].abs())[:, 0]
    return out, lse, size


def reserve(table, uses, lengths, counts, tokens, slots):
    """Lists in, lists out: the table, the uses, starts, the slot map, what was missing."""
    table, uses = [list(r) for r in table], list(uses)
    free = iter([p for p, u in enumerate(uses) if u == 0])
    starts, slot_map, missing = [0], [], 0
    for row, n, m in zip(table, lengths, counts):
        m = 0 if n < 0 or m < 0 else min(m, tokens - starts[-1])
        for c in range(n // slots, min(-(-(n + m) // slots), len(row))) if m else ():
            if not 0 <= row[c] < len(uses):
                page = next(free, None)
                if page is None:
                    missing += 1
                else:
                    row[c], uses[page] = page, 1
        starts.append(starts[-1] + m)
        for i in range(n, n + m):
            page = row[i // slots] if i // slots < len(row) else -1
            slot_map.append(page * slots + i % slots if 0 <= page < len(uses) else -1)
    return table, uses, starts, slot_map + [-1] * (tokens - len(slot_map)), missing
