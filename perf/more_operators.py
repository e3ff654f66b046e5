"""The library's operators for keys and values that come from one latent vector a token, as cases to be timed: attention over
keys that are part per head and part shared by all heads (training, prompts), attention over a cache of the latent rows
themselves (serving), and what a batch needs before it: pages for its new rows, and the rows in them.

`run` makes one pass: with `own` through the library's entry points, else in plain torch operations (32 bits, rounded
once at the end).  `exact` computes the same results in 64 bits in another way.

Kinds of cases
  step      forward and backward of causal attention with a shared part of the keys; `packed`: sequences of different lengths in one row
  prompt    its forward alone: a prompt, or with fewer queries than keys a chunk of one
  absorb    new tokens of every sequence over the cache of latent rows: one each (decoding), or `mixed` with chunks of prompts
  reserve   a step of a serving engine's bookkeeping: some sequences have ended, all get pages for their new rows and the rows their slots
  rows      packed rows go to their slots: latent rows, or with `hk` keys and values of that many heads
"""
import math
import random

import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}


def listed():
    return [
        # the smallest training call: a few short sequences of odd length, narrow heads
        dict(name='step_small', kind='step', dtype='fp16', b=2, h=4, sq=331, sk=331, e=64, r=32, ev=64),
        # training on one long sequence, the largest
        dict(name='step_long', kind='step', dtype='bf16', b=1, h=16, sq=8192, sk=8192, e=128, r=64, ev=128),
        # training on packed sequences of very different lengths
        dict(name='step_packed', kind='step', dtype='bf16', b=12, h=16, sq=4000, sk=4000, e=128, r=64, ev=128, packed=True),
        # a chunk of a long prompt behind what came before it
        dict(name='prompt_chunk', kind='prompt', dtype='fp16', b=1, h=16, sq=4096, sk=20011, e=128, r=64, ev=128),
        # decoding one sequence with the heads that one of several cards has: latency
        dict(name='absorb_one', kind='absorb', dtype='bf16', b=1, hq=16, length=4096, e=576, ev=512, page=64),
        # decoding a batch, all heads on one card
        dict(name='absorb_many', kind='absorb', dtype='bf16', b=64, hq=128, length=8192, e=576, ev=512, page=64, ragged=True),
        # decoding a batch with few heads a card: the cache's bytes
        dict(name='absorb_narrow', kind='absorb', dtype='fp16', b=48, hq=16, length=16384, e=576, ev=512, page=16, ragged=True),
        # a batch in which some sequences decode and some read chunks of their prompts
        dict(name='absorb_mixed', kind='absorb', dtype='bf16', b=24, hq=32, length=6000, e=576, ev=512, page=32, ragged=True, mixed=400),
        # the bookkeeping of a decoding step, a few of whose sequences are new
        dict(name='reserve_step', kind='reserve', b=200, length=4096, page=64, pool=16384, mixed=900),
        # the same for a large pool and long prompts
        dict(name='reserve_prompts', kind='reserve', b=500, length=6000, page=16, pool=400000, mixed=6000),
        # a decoding step's latent rows
        dict(name='rows_step', kind='rows', dtype='bf16', tokens=200, e=576, page=64, pool=700),
        # prompts' keys and values
        dict(name='rows_prompts', kind='rows', dtype='fp16', tokens=30011, e=128, hk=8, page=16, pool=2500),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['step', 'step', 'prompt', 'absorb', 'absorb', 'absorb', 'reserve', 'rows'])
    c = dict(kind=kind)
    if kind != 'reserve':
        c['dtype'] = rng.choice(['bf16', 'fp16'])
    if kind in ('step', 'prompt'):
        c['e'], c['r'], c['ev'] = rng.choice([(128, 64, 128), (128, 64, 128), (128, 32, 128), (96, 32, 96), (64, 64, 64), (64, 32, 64), (40, 24, 56)])
        c['h'] = rng.choice([1, 3, 4, 8, 16])
        c['packed'] = kind == 'step' and rng.random() < 0.4
        c['b'] = rng.randint(2, 12) if c['packed'] else _log(rng, 1, 6)
        c['sq'] = _log(rng, 1, max(64, min(6000, 8192 * 16 // (c['b'] * c['h']))))
        c['sk'] = c['sq'] + (_log(rng, 1, 8192) if kind == 'prompt' else 0)
    elif kind == 'absorb':
        c['e'], c['ev'] = rng.choice([(576, 512), (576, 512), (544, 512), (320, 256), (288, 256), (136, 128)])
        c['hq'] = rng.choice([1, 4, 8, 16, 20, 32, 64, 128])
        c['page'] = rng.choice([16, 32, 64, 256])
        c['b'] = _log(rng, 1, 64)
        c['length'] = _log(rng, 1, 16384 if c['b'] * c['hq'] <= 1024 else 6000)
        c['ragged'] = rng.random() < 0.7
        if rng.random() < 0.4:
            c['mixed'] = _log(rng, 2, 300 if c['hq'] <= 32 else 60)
    elif kind == 'reserve':
        c['b'], c['length'], c['page'] = _log(rng, 1, 600), _log(rng, 1, 8000), rng.choice([16, 32, 64, 256])
        c['mixed'] = _log(rng, 1, 4000)
        # room for what the sequences hold, and for some, most or all of what they ask for
        c['pool'] = max(1, int(_held(c) + _wanted(c) * rng.choice([0.7, 1.0, 1.3, 4.0, 16.0])))
    else:
        c['page'], c['tokens'] = rng.choice([16, 64]), _log(rng, 1, 30000)
        if rng.random() < 0.5:
            c['hk'], c['e'] = rng.choice([1, 4, 8]), rng.choice([64, 128, 256])
        else:
            c['e'] = rng.choice([136, 320, 576])
        c['pool'] = -(-c['tokens'] // c['page']) + rng.randint(1, 600)
    return c


# ---- what a case's numbers stand for --------------------------------------------------------------------------

def _lengths(case):
    """Tokens of every sequence: all alike, or spread over the range up to the longest (which is among them)."""
    top = case['sq'] if case['kind'] in ('step', 'prompt') else case['length']
    n = case['b']
    if not (case.get('packed') or case.get('ragged') or case['kind'] == 'reserve'):
        return [top] * n
    rng = random.Random(top * 131 + n)
    lens = [top] + [_log(rng, max(1, top // 24), top) for _ in range(n - 1)]
    rng.shuffle(lens)
    return lens


def _batch(case):
    """Filled slots and new tokens of every sequence: one token, or of some the chunk of a prompt, whose first chunk it may be."""
    lens = _lengths(case)
    if not case.get('mixed'):
        return lens, [1] * len(lens)
    rng = random.Random(case['mixed'] * 17 + len(lens))
    counts = [1] * len(lens)
    for z in range(len(lens)):
        if rng.random() < 0.2 or z == 0:
            counts[z] = _log(rng, 1, case['mixed']) if z else case['mixed']
            lens[z] = 0 if rng.random() < 0.5 or case['kind'] == 'reserve' else lens[z]
    return lens, counts


def _pages(n, page):
    return -(-n // page)


def _held(case):
    lens, _ = _batch(case)
    return sum(_pages(n, case['page']) for n in lens)


def _wanted(case):
    return sum(_pages(n + m, case['page']) - _pages(n, case['page']) for n, m in zip(*_batch(case)))


def _pairs(sq, sk):
    """(query, key) pairs of one sequence and head under the causal mask, queries at the last keys."""
    return sq * (sk - sq) + sq * (sq + 1) // 2


def work(case):
    kind = case['kind']
    if kind in ('step', 'prompt'):
        lens = _lengths(case)
        extra = case['sk'] - case['sq']
        e, r, ev, h = case['e'], case['r'], case['ev'], case['h']
        pairs = sum(_pairs(n, n + extra) for n in lens)
        rows_q, rows_k = sum(lens), sum(n + extra for n in lens)
        # forward: query, key, value, shared key in, out out.  A step: the gradient in as well, four gradients out
        q, k, o = rows_q * h * (e + r), rows_k * (h * (e + ev) + r), rows_q * h * ev
        if kind == 'prompt':
            return {'bytes': 2 * (q + k + o), 'flops': 2 * (e + r + ev) * pairs * h}
        return {'bytes': 2 * (2 * q + 2 * k + 2 * o), 'flops': 2 * (4 * (e + r) + 3 * ev) * pairs * h}
    if kind == 'absorb':
        lens, counts = _batch(case)
        rows, e, ev = sum(counts) * case['hq'], case['e'], case['ev']
        slots = sum(n + m for n, m in zip(lens, counts))
        pairs = sum(_pairs(m, n + m) for n, m in zip(lens, counts))
        return {'bytes': 2 * (e * slots + (e + ev) * rows), 'flops': 2 * (e + ev) * pairs * case['hq']}
    if kind == 'reserve':
        # uses, lengths, counts and the columns in question in; offsets, slots, pages and their uses out
        return {'bytes': 4 * case['pool'] + 12 * case['b'] + 8 * sum(_batch(case)[1]) + 12 * _wanted(case), 'flops': 0}
    return {'bytes': case['tokens'] * (8 + 2 * 2 * case['e'] * (2 * case['hk'] if 'hk' in case else 1)), 'flops': 0}


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    kind = case['kind']
    dt = _DTYPES[case.get('dtype', 'bf16')]

    def randn(*shape):
        return torch.randn(*shape, device='cuda', dtype=torch.float32, generator=gen).to(dt)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device='cuda')

    def offsets(counts):
        off = [0]
        for n in counts:
            off.append(off[-1] + n)
        return off

    s = dict(case=case)
    if kind in ('step', 'prompt'):
        h, e, r, ev = case['h'], case['e'], case['r'], case['ev']
        s['scale'] = 1.0 / math.sqrt(e + r)
        lens = _lengths(case)
        if case.get('packed'):
            off = offsets(lens)
            b, sq, sk = 1, off[-1], off[-1]
            s.update(offsets=off, cu=ints(off), longest=max(lens))
        else:
            b, sq, sk = case['b'], case['sq'], case['sk']
        # tensors as projections leave them: (batch, tokens, heads, columns) in memory, keys and values of a token's head side by side
        s['q'] = randn(b, sq, h, e + r).transpose(1, 2)
        kv = randn(b, sk, h, e + ev).transpose(1, 2)
        s['k'], s['v'], s['shared'] = kv[..., :e], kv[..., e:], randn(b, sk, r)
        if kind == 'step':
            s['dout'] = randn(b, sq, h, ev).transpose(1, 2)
            for n in ('q', 'k', 'v', 'shared'):
                s[n] = s[n].detach().requires_grad_(True)
        return s
    page = case['page']
    if kind == 'absorb':
        lens, counts = _batch(case)
        e, off = case['e'], offsets(counts)
        need = [_pages(n + m, page) for n, m in zip(lens, counts)]
        # a pool with some pages that belong to nobody; a sequence's pages lie anywhere in it
        total = sum(need) + 7
        order = torch.randperm(total, device='cuda', generator=gen).to(torch.int32).tolist()
        table, at = [], 0
        for n in need:
            table.append(order[at:at + n] + [-1] * (max(need) - n))
            at += n
        # (the scores' scale is that of the heads that the queries come from, a third as wide as the latent rows)
        s.update(table=ints(table), lengths=ints(lens), starts=ints(off), offsets=off, longest=max(lens), scale=math.sqrt(3.0 / e))
        s['cache'] = randn(total, 1, page, e)
        s['q'] = randn(off[-1], case['hq'], e)
        return s
    if kind == 'reserve':
        lens, counts = _batch(case)
        pool = case['pool']
        columns = max(_pages(n + m, page) for n, m in zip(lens, counts)) + 2
        order = torch.randperm(pool, device='cuda', generator=gen).tolist()
        table, at = [[-1] * columns for _ in lens], 0
        for z, n in enumerate(lens):
            for c in range(_pages(n, page)):
                table[z][c] = order[at]
                at += 1
        # those that begin anew stand where others have ended, whose pages are still theirs
        for z, n in enumerate(lens):
            for c in range(min(columns, (pool - at) // 64) if n == 0 else 0):
                table[z][c] = order[at]
                at += 1
        uses = torch.zeros(pool, dtype=torch.int32, device='cuda')
        uses[torch.tensor(order[:at], dtype=torch.int64, device='cuda')] = 1
        b = len(lens)
        s.update(table=ints(table), uses=uses, lengths=ints(lens), counts=ints(counts), tokens=sum(counts), sequences=ints(list(range(b))),
                 first=ints([_pages(n, page) for n in lens]), last=ints([columns] * b))
        return s
    n, pool = case['tokens'], case['pool']
    # runs of slots in pages that lie anywhere, a few rows without a place
    order = torch.randperm(pool, device='cuda', generator=gen)
    i = torch.arange(n, device='cuda')
    slot = order[i // page] * page + i % page
    s['slots'] = torch.where(torch.rand(n, device='cuda', generator=gen) < 0.01, torch.full_like(slot, -1), slot)
    e = case['e']
    if 'hk' in case:
        for name in 'kv':
            s[name] = randn(n, case['hk'], e)
            s[name + '_cache'] = randn(pool, page, case['hk'], e).transpose(1, 2)
    else:
        s.update(k=randn(n, 1, e), k_cache=randn(pool, 1, page, e), v=None, v_cache=None)
    return s


# ---- the library's operators ----------------------------------------------------------------------------------

def _run_own(s):
    from aotriton_amd import cache, torch_ops
    c, kind = s['case'], s['case']['kind']
    if kind in ('step', 'prompt'):
        packed = {}
        if c.get('packed'):
            packed = dict(cu_seqlens_q=s['cu'], cu_seqlens_k=s['cu'], max_seqlen_q=s['longest'], max_seqlen_k=s['longest'])
        out = torch_ops.latent_attention(s['q'], s['k'], s['v'], s['shared'], scale=s['scale'], **packed)
        if kind == 'prompt':
            return out
        return (out.detach(), *torch.autograd.grad(out, (s['q'], s['k'], s['v'], s['shared']), s['dout']))
    if kind == 'absorb':
        return cache.latent_attention(s['q'], s['cache'], s['table'], s['lengths'], s['starts'], c['ev'], s['scale'], max_length=s['longest'])
    if kind == 'reserve':
        cache.free(s['table'], s['uses'], s['sequences'], s['first'], s['last'])
        starts, slots, missing = cache.reserve(s['table'], s['uses'], s['lengths'], s['counts'], s['tokens'], c['page'])
        return starts, slots, missing, s['table'], s['uses']
    cache.append_packed(s['k'], s['v'], s['k_cache'], s['v_cache'], s['slots'])
    return s['k_cache'] if s['v'] is None else (s['k_cache'], s['v_cache'])


# ---- the same in plain operations -----------------------------------------------------------------------------

def _plain_expanded(q, k, v, shared, dout, scale, block=1024):
    """(heads, rows, columns) of one sequence, shared (rows, columns); block after block of queries.  Returns out, and with dout
    the gradients."""
    h, sq, _ = q.shape
    sk, e = k.shape[1:]
    q, v = q.float(), v.float()
    keys = torch.cat([k.float(), shared.float()[None].expand(h, -1, -1)], 2)
    out = torch.zeros(h, sq, v.shape[2], device=q.device)
    if dout is not None:
        dout = dout.float()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(keys), torch.zeros_like(v)
    for r0 in range(0, sq, block):
        r1 = min(r0 + block, sq)
        n = r1 + sk - sq
        if n <= 0:
            continue
        hidden = torch.arange(n, device=q.device)[None] > torch.arange(r0, r1, device=q.device)[:, None] + sk - sq
        qb, kb, vb = q[:, r0:r1], keys[:, :n], v[:, :n]
        x = torch.matmul(qb, kb.transpose(1, 2)).mul_(scale).masked_fill_(hidden[None], -math.inf)
        top = x.amax(2, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        x = x.sub_(top).exp_()
        x = x.div_(x.sum(2, keepdim=True).clamp(min=1e-30))
        o = torch.matmul(x, vb)
        out[:, r0:r1] = o
        if dout is None:
            continue
        do = dout[:, r0:r1]
        dv[:, :n] += torch.matmul(x.transpose(1, 2), do)
        ds = torch.matmul(do, vb.transpose(1, 2))
        ds = ds.sub_((do * o).sum(2, keepdim=True)).mul_(x).mul_(scale)
        dq[:, r0:r1] = torch.matmul(ds, kb)
        dk[:, :n] += torch.matmul(ds.transpose(1, 2), qb)
    return out if dout is None else (out, dq, dk[..., :e], dv, dk[..., e:].sum(0))


def _per_sequence(s, f):
    """f over the parts of every sequence, put together in the layout of the inputs."""
    c = s['case']
    names = ['q', 'k', 'v', 'shared'] + (['dout'] if c['kind'] == 'step' else [])
    t = {n: s[n].detach() for n in names}
    if c.get('packed'):
        # (the rows of a sequence are the last but one dimension of its tensors)
        parts = [f(*(t[n][0][..., a:z, :] for n in names)) for a, z in zip(s['offsets'], s['offsets'][1:])]
        join = lambda xs: torch.cat(list(xs), -2)[None]
    else:
        parts = [f(*(t[n][i] for n in names)) for i in range(c['b'])]
        join = lambda xs: torch.stack(list(xs))
    if c['kind'] == 'prompt':
        return join(parts)
    return tuple(join(x) for x in zip(*parts))


def _plain_absorbed(q, rows, first, scale, ev):
    """q (sequences, tokens, heads, columns) at positions first + token of rows (sequences, slots, columns)."""
    b, t, h, e = q.shape
    n = torch.arange(rows.shape[1], device=q.device)
    seen = n[None, None] <= first[:, None, None] + torch.arange(t, device=q.device)[None, :, None]
    x = torch.matmul(q.float().view(b, t * h, e), rows.transpose(1, 2)).mul_(scale).view(b, t, h, -1)
    x = x.masked_fill_(~seen[:, :, None], -math.inf)
    x = x.sub_(x.amax(3, keepdim=True)).exp_()
    x = x.div_(x.sum(3, keepdim=True))
    return torch.matmul(x.view(b, t * h, -1), rows[..., :ev]).view(b, t, h, ev)


def _plain_absorb(s):
    c, q = s['case'], s['q']
    lens, counts = _batch(c)
    page, e, ev = c['page'], c['e'], c['ev']
    table, lengths = s['table'].long().clamp(min=0), s['lengths'].long()
    one = [z for z, m in enumerate(counts) if m == 1]
    out = torch.empty(*q.shape[:2], ev, device=q.device)
    # the sequences with one token together, as many as keeps them small; the others one by one
    for i in range(0, len(one), 32):
        some = one[i:i + 32]
        at = torch.tensor(some, device=q.device)
        columns = _pages(max(lens[z] for z in some) + 1, page)
        rows = s['cache'][table[at, :columns]].view(len(some), columns * page, e).float()
        where = s['starts'].long()[at]
        out[where] = _plain_absorbed(q[where][:, None], rows, lengths[at], s['scale'], ev)[:, 0]
    for z, m in enumerate(counts):
        if m > 1:
            rows = s['cache'][table[z, :_pages(lens[z] + m, page)]].view(1, -1, e).float()
            a = s['offsets'][z]
            out[a:a + m] = _plain_absorbed(q[None, a:a + m], rows, lengths[z:z + 1], s['scale'], ev)[0]
    return out.to(q.dtype)


def _plain_reserve(s):
    table, uses, page, n = s['table'], s['uses'], s['case']['page'], s['tokens']
    columns, pool = table.shape[1], uses.shape[0]
    # what stands behind the filled columns goes
    c = torch.arange(columns, device='cuda')[None]
    gone = (c >= s['first'][:, None]) & (c < s['last'][:, None])
    pages = table.long()
    there = gone & (pages >= 0) & (pages < pool)
    uses.index_add_(0, pages.clamp(0, pool - 1).flatten(), -there.flatten().to(torch.int32))
    table.masked_fill_(gone, -1)
    # pages for the new rows, the first free ones in the order of sequences and columns
    lengths, counts = s['lengths'].long(), s['counts'].long()
    ends = counts.cumsum(0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    want = (c >= (lengths // page)[:, None]) & (c * page < (lengths + counts)[:, None]) & (counts > 0)[:, None]
    want &= (table < 0) | (table >= pool)
    rank = want.flatten().cumsum(0) - 1
    free = uses == 0
    order = torch.argsort((~free).to(torch.int8), stable=True)
    got = want & (rank.view_as(want) < free.sum())
    page_of = order[rank.clamp(0, pool - 1)].view_as(want)
    table.copy_(torch.where(got, page_of.to(torch.int32), table))
    uses.index_add_(0, page_of.flatten(), got.flatten().to(torch.int32))
    missing = (want & ~got).sum().to(torch.int32).view(1)
    i = torch.arange(n, device='cuda')
    z = torch.searchsorted(ends, i, right=True)
    slot = lengths[z] + i - starts[z]
    at = table[z, slot // page].long()
    return starts.to(torch.int32), torch.where(at >= 0, at * page + slot % page, torch.full_like(at, -1)), missing, table, uses


def _run_plain(s):
    c, kind = s['case'], s['case']['kind']
    if kind in ('step', 'prompt'):
        def f(q, k, v, shared, dout=None):
            r = _plain_expanded(q, k, v, shared, dout, s['scale'])
            return r.to(q.dtype) if dout is None else tuple(x.to(q.dtype) for x in r)
        return _per_sequence(s, f)
    if kind == 'absorb':
        return _plain_absorb(s)
    if kind == 'reserve':
        return _plain_reserve(s)
    page = c['page']
    here = s['slots'] >= 0
    slots = s['slots'][here]
    for new, kept in ((s['k'], s['k_cache']), (s['v'], s['v_cache'])):
        if new is not None:
            kept.transpose(1, 2)[slots // page, slots % page] = new[here]
    return s['k_cache'] if s['v'] is None else (s['k_cache'], s['v_cache'])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- in 64 bits, another way ------------------------------------------------------------------------------------

def _exact_expanded(q, k, v, shared, dout, scale):
    """Head by head, the scores as the sum of two products, band by band of queries over all keys."""
    h, sq, _ = q.shape
    sk, e = k.shape[1:]
    c = shared.double()
    outs, dqs, dks, dvs = [], [], [], []
    dc = torch.zeros_like(c)
    for i in range(h):
        kd, vd = k[i].double(), v[i].double()
        o_h, dq_h, dk_h, dv_h = [], [], torch.zeros_like(kd), torch.zeros_like(vd)
        for r0 in range(0, sq, 2048):
            qd = q[i, r0:r0 + 2048].double()
            seen = torch.ones(len(qd), sk, dtype=torch.bool, device=q.device).tril(r0 + sk - sq)
            x = torch.where(seen, (qd[:, :e] @ kd.T + qd[:, e:] @ c.T) * scale, -torch.inf)
            p = torch.where(seen, torch.exp(x - torch.logsumexp(x, 1, keepdim=True)), 0.0)
            o_h.append(p @ vd)
            if dout is None:
                continue
            do = dout[i, r0:r0 + 2048].double()
            dv_h += p.T @ do
            dp = do @ vd.T
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
            dq_h.append(torch.cat([ds @ kd, ds @ c], 1))
            dk_h += ds.T @ qd[:, :e]
            dc += ds.T @ qd[:, e:]
        outs.append(torch.cat(o_h))
        if dout is not None:
            dqs.append(torch.cat(dq_h))
            dks.append(dk_h)
            dvs.append(dv_h)
    if dout is None:
        return torch.stack(outs)
    return torch.stack(outs), torch.stack(dqs), torch.stack(dks), torch.stack(dvs), dc


def _exact_absorb(s):
    c, q = s['case'], s['q']
    out = torch.empty(*q.shape[:2], c['ev'], dtype=torch.float64, device='cuda')
    table = s['table'].tolist()
    for z, (n, m) in enumerate(zip(*_batch(c))):
        order = torch.tensor(table[z][:_pages(n + m, c['page'])], device='cuda')
        x = s['cache'][order, 0].reshape(-1, c['e'])[:n + m].double()
        for t in range(0, m, 64):
            a = s['offsets'][z] + t
            qd = q[a:a + min(64, m - t)].double()
            p = torch.einsum('thc,nc->htn', qd, x) * s['scale']
            hidden = torch.arange(n + m, device='cuda')[None] > n + t + torch.arange(len(qd), device='cuda')[:, None]
            p = torch.softmax(p.masked_fill(hidden[None], -torch.inf), 2)
            out[a:a + len(qd)] = torch.einsum('htn,nc->thc', p, x[:, :c['ev']])
    return out


def _exact_reserve(s):
    page = s['case']['page']
    table, uses = s['table'].tolist(), s['uses'].tolist()
    lens, counts = s['lengths'].tolist(), s['counts'].tolist()
    for row, a, z in zip(table, s['first'].tolist(), s['last'].tolist()):
        for c in range(a, z):
            if row[c] >= 0:
                uses[row[c]] -= 1
            row[c] = -1
    free = iter([p for p, u in enumerate(uses) if u == 0])
    starts, slots, missing = [0], [], 0
    for row, n, m in zip(table, lens, counts):
        for c in range(n // page, _pages(n + m, page) if m else 0):
            if row[c] < 0:
                row[c] = next(free, -1)
                if row[c] >= 0:
                    uses[row[c]] += 1
                else:
                    missing += 1
        starts.append(starts[-1] + m)
        slots += [row[i // page] * page + i % page if row[i // page] >= 0 else -1 for i in range(n, n + m)]
    as_ints = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device='cuda')
    return as_ints(starts), as_ints(slots, torch.int64), as_ints([missing]), as_ints(table), as_ints(uses)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case['kind']
    if kind in ('step', 'prompt'):
        return _per_sequence(s, lambda q, k, v, shared, dout=None: _exact_expanded(q, k, v, shared, dout, s['scale']))
    if kind == 'absorb':
        return _exact_absorb(s)
    if kind == 'reserve':
        return _exact_reserve(s)
    here = s['slots'] >= 0
    page, slot = s['slots'][here] // case['page'], s['slots'][here] % case['page']
    outs = []
    for new, kept in ((s['k'], s['k_cache']), (s['v'], s['v_cache'])):
        if new is not None:
            x = kept.double()
            for h in range(x.shape[1]):
                x[page, h, slot] = new[here, h].double()
            outs.append(x)
    return outs[0] if s['v'] is None else tuple(outs)
