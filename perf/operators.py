"""The library's operators for long contexts and for serving, as cases to be timed: attention with a sliding
window and first tokens that stay visible, attention for a tree of drafted tokens over a cache of pages, and the
pages of that cache.

`run` makes one pass: with `own` through the library's entry points, else in plain torch operations (32 bits, rounded
once at the end).  `exact` computes the same results in 64 bits in another way.

Kinds of cases
  step      forward and backward of windowed attention (training); `packed`: sequences of different lengths in one row
  prompt    its forward alone: a prompt, or with fewer queries than keys a chunk of one
  tree      drafted tokens over a cache of pages; one token is plain decoding
  append    drafted rows go into their pages and the accepted path of the tree moves together
  beam      sequences are freed and others forked into their place
  copy      whole pages
"""
import math
import random

import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}


def listed():
    return [
        # the smallest training call: a few short sequences of odd length
        dict(name='step_small', kind='step', dtype='fp16', b=2, hq=4, hk=2, sq=331, sk=331, d=64, window=100, sinks=4),
        # training on long sequences, grouped heads
        dict(name='step_long', kind='step', dtype='bf16', b=1, hq=32, hk=8, sq=8192, sk=8192, d=128, window=1024, sinks=4),
        # training on packed sequences of very different lengths
        dict(name='step_packed', kind='step', dtype='bf16', b=16, hq=16, hk=4, sq=6000, sk=6000, d=128, window=512, sinks=17,
             packed=True),
        # a long prompt read at once, the largest
        dict(name='prompt_long', kind='prompt', dtype='bf16', b=1, hq=32, hk=8, sq=32768, sk=32768, d=128, window=4096, sinks=64),
        # a serving engine's prompt chunk behind what came before it, narrow heads
        dict(name='prompt_chunk', kind='prompt', dtype='fp16', b=4, hq=16, hk=16, sq=512, sk=4601, d=64, window=2048, sinks=8),
        # one sequence, one token: latency
        dict(name='tree_one', kind='tree', dtype='bf16', b=1, hq=32, hk=8, t=1, length=4096, d=128, page=64, window=0, sinks=0),
        # decoding of a large batch with different lengths: the cache's bytes
        dict(name='tree_batch', kind='tree', dtype='bf16', b=64, hq=32, hk=8, t=1, length=8192, d=128, page=16, window=0, sinks=0,
             ragged=True),
        # drafted trees over long caches
        dict(name='tree_drafts', kind='tree', dtype='fp16', b=8, hq=32, hk=8, t=48, length=16384, d=128, page=64, window=0, sinks=0,
             ragged=True),
        # the windowed model's drafts: the cache is long, what is visible of it short
        dict(name='tree_window', kind='tree', dtype='bf16', b=32, hq=16, hk=2, t=7, length=16384, d=64, page=32, window=1024, sinks=4,
             ragged=True),
        # drafted rows into their pages, and the accepted ones together
        dict(name='append', kind='append', dtype='bf16', b=32, hk=8, t=24, length=2048, d=128, page=64),
        # beam search: the losing sequences go, the winning ones are forked
        dict(name='beam', kind='beam', dtype='fp16', b=16, hk=8, length=4000, d=128, page=64),
        # pages moved in bulk
        dict(name='copy', kind='copy', dtype='bf16', b=2048, hk=8, d=128, page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['step', 'step', 'prompt', 'tree', 'tree', 'tree', 'append', 'beam', 'copy'])
    c = dict(kind=kind, dtype=rng.choice(['bf16', 'fp16']))
    if kind in ('step', 'prompt'):
        c['d'] = rng.choice([64, 80, 96, 128])
        c['hk'] = rng.choice([1, 2, 4, 8])
        c['hq'] = c['hk'] * rng.choice([1, 2, 4])
        c['packed'] = rng.random() < 0.4
        c['b'] = rng.randint(2, 12) if c['packed'] else _log(rng, 1, 8)
        top = 8192 if kind == 'step' else 16384
        c['sq'] = _log(rng, 64, max(64, min(top, top * 32 // (c['b'] * c['hq']))))
        c['sk'] = c['sq'] + (_log(rng, 1, 4096) if kind == 'prompt' and not c['packed'] and rng.random() < 0.4 else 0)
        c['window'] = _log(rng, 16, 2048)
        c['sinks'] = rng.choice([0, 1, 4, 4, 16, 40, 64, 128])
    elif kind == 'tree':
        c['d'] = rng.choice([64, 128])
        c['hk'] = rng.choice([1, 2, 8])
        c['hq'] = c['hk'] * rng.choice([1, 4, 7, 8])
        c['t'] = rng.choice([1, 1, _log(rng, 2, 64)])
        c['page'] = rng.choice([16, 32, 64, 256])
        c['b'] = _log(rng, 1, 48)
        c['length'] = _log(rng, 1, 16384 if c['b'] <= 16 else 6000)
        c['window'], c['sinks'] = (_log(rng, 16, 2048), rng.choice([0, 4, 33])) if rng.random() < 0.4 else (0, 0)
        c['ragged'] = rng.random() < 0.7
    elif kind == 'copy':
        c['b'], c['hk'], c['d'], c['page'] = _log(rng, 8, 2048), rng.choice([1, 4, 8]), rng.choice([64, 128]), rng.choice([16, 64])
    else:
        c['hk'], c['d'], c['page'] = rng.choice([1, 4, 8]), rng.choice([64, 128]), rng.choice([16, 32, 64])
        c['b'] = _log(rng, 1, 32) if kind == 'append' else _log(rng, 1, 16)
        c['length'] = _log(rng, 1, 2048 if kind == 'append' else 4000)
        if kind == 'append':
            c['t'] = _log(rng, 1, 64)
    return c


# ---- what a case's numbers stand for --------------------------------------------------------------------------

def _lengths(case):
    """Tokens of every sequence: all alike, or spread over the range up to the longest (which is among them)."""
    top = case['sq'] if case['kind'] in ('step', 'prompt') else case['length']
    n = case['b']
    if not (case.get('packed') or case.get('ragged')):
        return [top] * n
    rng = random.Random(top * 131 + n)
    lens = [top] + [_log(rng, max(1, top // 24), top) for _ in range(n - 1)]
    rng.shuffle(lens)
    return lens


def _visible_pairs(sq, sk, window, sinks):
    """(query, key) pairs of one sequence and head."""
    p = torch.arange(sq, dtype=torch.int64) + (sk - sq)
    lo = (p - window + 1).clamp(min=0)
    seen = (p + 1 - lo).clamp(min=0) + torch.minimum(lo, torch.full_like(lo, sinks)) * (p >= 0)
    return int(seen.sum())


def work(case):
    d, kind = case['d'], case['kind']
    if kind in ('step', 'prompt'):
        lens = _lengths(case)
        extra = case['sk'] - case['sq']
        pairs = sum(_visible_pairs(n, n + extra, case['window'], case['sinks']) for n in lens)
        rows_q, rows_k = sum(lens) * case['hq'], sum(n + extra for n in lens) * case['hk']
        # forward: q, k, v in, out out.  A step: q, k, v, dout in, out, dq, dk, dv out
        step = kind == 'step'
        return {'bytes': 2 * d * ((4 if step else 2) * rows_q + (4 if step else 2) * rows_k),
                'flops': (14 if step else 4) * d * pairs * case['hq']}
    if kind == 'tree':
        slots = 0
        for n in _lengths(case):
            seen = n if not case['window'] else min(n, case['window'] + min(case['sinks'], max(n - case['window'], 0)))
            slots += seen + case['t']
        rows = case['b'] * case['t'] * case['hq']
        return {'bytes': 2 * d * (2 * slots * case['hk'] + 2 * rows), 'flops': 4 * d * slots * case['t'] * case['hq']}
    row = 2 * d * case['hk'] * 2          # K and V of a token
    if kind == 'append':
        kept = _kept(case)
        return {'bytes': 2 * row * case['b'] * (case['t'] + kept), 'flops': 0}
    if kind == 'beam':
        pages = -(-case['length'] // case['page'])
        tail = case['page'] if case['length'] % case['page'] else 0
        return {'bytes': case['b'] * (2 * row * tail + 4 * 4 * pages), 'flops': 0}
    return {'bytes': 2 * row * case['b'] * case['page'], 'flops': 0}


def _kept(case):
    return max(1, case['t'] // 4)


def _tree(rng, t):
    """Parents of a drafted tree: every token behind an earlier one, mostly a late one."""
    return [-1 if i == 0 or rng.random() < 0.1 else i - 1 - min(i - 1, int(rng.expovariate(0.5))) for i in range(t)]


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    host = random.Random(seed)
    dt, d = _DTYPES[case['dtype']], case['d']

    def randn(*shape):
        return torch.randn(*shape, device='cuda', dtype=torch.float32, generator=gen).to(dt)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device='cuda')

    s = dict(case=case, scale=1.0 / math.sqrt(d))
    if case['kind'] in ('step', 'prompt'):
        lens = _lengths(case)
        hq, hk = case['hq'], case['hk']
        # tensors as projections leave them: (batch, tokens, heads, head dim) in memory
        if case.get('packed'):
            b, sq, sk = 1, sum(lens), sum(lens)
            off = [0]
            for n in lens:
                off.append(off[-1] + n)
            s.update(offsets=off, cu=ints(off), longest=max(lens))
        else:
            b, sq, sk = case['b'], case['sq'], case['sk']
        s['q'] = randn(b, sq, hq, d).transpose(1, 2)
        s['k'] = randn(b, sk, hk, d).transpose(1, 2)
        s['v'] = randn(b, sk, hk, d).transpose(1, 2)
        if case['kind'] == 'step':
            s['dout'] = randn(b, sq, hq, d).transpose(1, 2)
            for n in 'qkv':
                s[n].requires_grad_(True)
        return s

    hk, page = case['hk'], case['page']
    if case['kind'] == 'copy':
        n = case['b']
        s['k_cache'], s['v_cache'] = randn(2 * n, hk, page, d), randn(2 * n, hk, page, d)
        order = torch.randperm(2 * n, device='cuda', generator=gen).to(torch.int32)
        s['source'], s['target'] = order[:n].contiguous(), order[n:].contiguous()
        return s

    lens = _lengths(case)
    t = case.get('t', 0)
    slots = -(-(max(lens) + t) // page)
    need = [-(-(n + t) // page) for n in lens]
    b = case['b']
    if case['kind'] == 'beam':
        # sequence i is the winner, b + i the loser that it replaces: both share all full pages already
        full, tail = divmod(lens[0], page)
        per = full + (2 if tail else 0)
        total = b * per
        order = torch.randperm(total, device='cuda', generator=gen).to(torch.int32).view(b, per)
        table = torch.full((2 * b, slots), -1, dtype=torch.int32, device='cuda')
        uses = torch.zeros(total, dtype=torch.int32, device='cuda')
        table[:b, :full] = order[:, :full]
        table[b:, :full] = order[:, :full]
        uses[order[:, :full].flatten().long()] = 2
        if tail:
            table[:b, full], table[b:, full] = order[:, full], order[:, full + 1]
            uses[order[:, full:].flatten().long()] = 1
        s.update(table=table, uses=uses, lengths=ints(lens * 2), source=ints(list(range(b))), target=ints(list(range(b, 2 * b))),
                 spare=order[:, per - 1].contiguous(), first=ints([0] * b), last=ints([slots] * b), full=full, tail=tail)
        s['k_cache'], s['v_cache'] = randn(total, hk, page, d), randn(total, hk, page, d)
        return s

    # a pool with some pages that belong to nobody; a sequence's pages lie anywhere in it
    total = sum(need) + 7
    order = torch.randperm(total, device='cuda', generator=gen).to(torch.int32).tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (slots - n))
        at += n
    s.update(table=ints(table), lengths=ints(lens), longest=max(lens))
    # a page's rows of one token lie together: (pages, slots, heads, head dim) in memory
    s['k_cache'] = randn(total, page, hk, d).transpose(1, 2)
    s['v_cache'] = randn(total, page, hk, d).transpose(1, 2)
    trees = [_tree(host, t) for _ in range(b)]
    s['parents'] = ints(trees) if t > 1 else None
    if case['kind'] == 'tree':
        s['q'] = randn(b, t, case['hq'], d).transpose(1, 2)
    else:
        s['k'], s['v'] = randn(b, t, hk, d).transpose(1, 2), randn(b, t, hk, d).transpose(1, 2)
        kept = _kept(case)
        s['path'] = ints([sorted(host.sample(range(t), kept)) for _ in range(b)])
        s['counts'] = ints([host.randint(1, kept) for _ in range(b)])
    return s


# ---- the library's operators ----------------------------------------------------------------------------------

def _run_own(s):
    from aotriton_amd import cache, torch_ops
    c, kind = s['case'], s['case']['kind']
    if kind in ('step', 'prompt'):
        packed = {}
        if c.get('packed'):
            packed = dict(cu_seqlens_q=s['cu'], cu_seqlens_k=s['cu'], max_seqlen_q=s['longest'], max_seqlen_k=s['longest'])
        out = torch_ops.sink_attention(s['q'], s['k'], s['v'], c['window'], c['sinks'], scale=s['scale'], **packed)
        if kind == 'prompt':
            return out
        return (out.detach(), *torch.autograd.grad(out, (s['q'], s['k'], s['v']), s['dout']))
    if kind == 'tree':
        return cache.tree_attention(s['q'], s['k_cache'], s['v_cache'], s['table'], s['lengths'], s['parents'],
                                    max_length=s['longest'], window=c['window'], sinks=c['sinks'], scale=s['scale'])
    if kind == 'append':
        cache.append(s['k'], s['v'], s['k_cache'], s['v_cache'], s['table'], s['lengths'])
        after = cache.keep_path(s['k_cache'], s['v_cache'], s['table'], s['lengths'], s['path'], s['counts'])
        return s['k_cache'], s['v_cache'], after
    if kind == 'beam':
        cache.free(s['table'], s['uses'], s['target'], s['first'], s['last'])
        cache.fork(s['k_cache'], s['v_cache'], s['table'], s['lengths'], s['uses'], s['source'], s['target'], s['spare'])
    else:
        cache.copy_pages(s['k_cache'], s['v_cache'], s['source'], s['target'])
        return s['k_cache'], s['v_cache']
    return s['k_cache'], s['v_cache'], s['table'], s['uses']


# ---- the same in plain operations -----------------------------------------------------------------------------

def _plain_attention(q, k, v, dout, window, sinks, scale, block=512):
    """(heads, rows, head dim) of one sequence, heads grouped; block after block of queries against the keys that any of
    them sees.  Returns out, and with dout the gradients."""
    hq, sq, d = q.shape
    hk, sk, _ = k.shape
    g, shift = hq // hk, sk - sq
    q, k, v = q.float(), k.float(), v.float()
    out = torch.zeros_like(q)
    if dout is not None:
        dout = dout.float()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for r0 in range(0, sq, block):
        r1 = min(r0 + block, sq)
        lo, hi = max(0, r0 + shift - window + 1), r1 + shift
        if hi <= 0:
            continue
        first = min(sinks, lo)
        keys = torch.cat([torch.arange(first, device=q.device), torch.arange(lo, hi, device=q.device)])
        p = torch.arange(r0, r1, device=q.device)[:, None] + shift
        seen = (keys[None] <= p) & ((keys[None] > p - window) | (keys[None] < sinks))
        hidden = ~seen.repeat(g, 1)[None]                             # (1, group * rows, keys)
        kb, vb = torch.cat([k[:, :first], k[:, lo:hi]], 1), torch.cat([v[:, :first], v[:, lo:hi]], 1)
        qb = q[:, r0:r1].reshape(hk, g * (r1 - r0), d)
        x = torch.matmul(qb, kb.transpose(1, 2)).mul_(scale).masked_fill_(hidden, -math.inf)
        top = x.amax(2, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        x = x.sub_(top).exp_()
        x = x.div_(x.sum(2, keepdim=True).clamp(min=1e-30))
        o = torch.matmul(x, vb)
        out[:, r0:r1] = o.view(hq, r1 - r0, d)
        if dout is None:
            continue
        do = dout[:, r0:r1].reshape(hk, g * (r1 - r0), d)
        ds = torch.matmul(do, vb.transpose(1, 2))
        ds = ds.sub_((do * o).sum(2, keepdim=True)).mul_(x).mul_(scale)
        dq[:, r0:r1] = torch.matmul(ds, kb).view(hq, r1 - r0, d)
        for grad, part in ((dk, torch.matmul(ds.transpose(1, 2), qb)), (dv, torch.matmul(x.transpose(1, 2), do))):
            grad[:, :first] += part[:, :first]
            grad[:, lo:hi] += part[:, first:]
    return out if dout is None else (out, dq, dk, dv)


def _per_sequence(s, f):
    """f over the (heads, rows, head dim) parts of every sequence, put together in the layout of the inputs."""
    c = s['case']
    names = ['q', 'k', 'v'] + (['dout'] if c['kind'] == 'step' else [])
    t = {n: s[n].detach() for n in names}
    if c.get('packed'):
        off = s['offsets']
        parts = [f(*(t[n][0, :, a:z] for n in names)) for a, z in zip(off, off[1:])]
        join = lambda xs: torch.cat(list(xs), 1)[None]
    else:
        parts = [f(*(t[n][i] for n in names)) for i in range(c['b'])]
        join = lambda xs: torch.stack(list(xs))
    if c['kind'] == 'prompt':
        return join(parts)
    return tuple(join(x) for x in zip(*parts))


def _plain_rows(s, t):
    """Page and slot in the page of the t rows behind every sequence's length."""
    page = s['k_cache'].shape[2]
    n = s['lengths'].long()[:, None] + torch.arange(t, device='cuda')
    return s['table'].long().gather(1, n // page), n % page


def _plain_tree(s):
    c = s['case']
    q, table, lengths = s['q'], s['table'].long(), s['lengths'].long()
    b, hq, t, d = q.shape
    pages, hk, page, _ = s['k_cache'].shape
    g = hq // hk
    n = torch.arange(table.shape[1] * page, device='cuda')
    if s['parents'] is None:
        kin = torch.eye(t, device='cuda').expand(b, t, t)
    else:
        step = (s['parents'].long()[:, :, None] == torch.arange(t, device='cuda')).float()
        kin = torch.eye(t, device='cuda') + step                      # the walk up to the root, twice as far each time
        for _ in range(6):
            step = torch.matmul(step, step)
            kin = kin + torch.matmul(kin, step)
    kin = kin > 0.5
    depth = kin.sum(2) - 1                                            # (b, t)
    draft = n[None] - lengths[:, None]                                # (b, slots): the drafted token in a slot
    is_draft = (draft >= 0) & (draft < t)
    at = draft.clamp(0, t - 1)
    seen = torch.where(is_draft[:, None], kin.gather(2, at[:, None].expand(b, t, -1)), (draft < 0)[:, None])
    if c['window']:
        where = torch.where(is_draft, lengths[:, None] + depth.gather(1, at), n[None])
        own_at = lengths[:, None] + depth
        seen = seen & ((where[:, None] > own_at[:, :, None] - c['window']) | (where[:, None] < c['sinks']))
    seen = seen[:, None, None]                                        # (b, 1, 1, t, slots)
    k, v = (x[table.clamp(min=0)].transpose(1, 2).reshape(b * hk, -1, d).float() for x in (s['k_cache'], s['v_cache']))
    x = torch.matmul(q.float().reshape(b * hk, g * t, d), k.transpose(1, 2)).mul_(s['scale']).view(b, hk, g, t, -1)
    x = x.masked_fill_(~seen, -math.inf)
    x = x.sub_(x.amax(4, keepdim=True)).exp_()
    x = x.div_(x.sum(4, keepdim=True))
    return torch.matmul(x.view(b * hk, g * t, -1), v).view(b, hq, t, d).to(q.dtype)


def _run_plain(s):
    c, kind = s['case'], s['case']['kind']
    if kind in ('step', 'prompt'):
        def f(q, k, v, dout=None):
            r = _plain_attention(q, k, v, dout, c['window'], c['sinks'], s['scale'])
            return r.to(q.dtype) if dout is None else tuple(x.to(q.dtype) for x in r)
        return _per_sequence(s, f)
    if kind == 'tree':
        return _plain_tree(s)
    caches = ('k_cache', 'v_cache')
    if kind == 'append':
        at, slot = _plain_rows(s, c['t'])
        for name, new in zip(caches, (s['k'], s['v'])):
            s[name].transpose(1, 2)[at, slot] = new.transpose(1, 2)
        i = torch.arange(s['path'].shape[1], device='cuda')
        live = i[None] < s['counts'][:, None]
        from_at, from_slot = at.gather(1, s['path'].long())[live], slot.gather(1, s['path'].long())[live]
        to_at, to_slot = at[:, :len(i)][live], slot[:, :len(i)][live]
        for name in caches:
            rows = s[name].transpose(1, 2)
            rows[to_at, to_slot] = rows[from_at, from_slot]
        return s['k_cache'], s['v_cache'], s['lengths'] + s['counts']
    if kind == 'beam':
        table, uses, target, source = s['table'], s['uses'], s['target'].long(), s['source'].long()
        gone = table[target].flatten()
        uses.index_add_(0, gone.clamp(min=0).long(), -(gone >= 0).to(torch.int32))
        rows = table[source]
        tails = rows[:, s['full']].long() if s['tail'] else None
        if s['tail']:
            rows[:, s['full']] = s['spare']
            for name in caches:
                s[name][s['spare'].long(), :, :s['tail']] = s[name][tails, :, :s['tail']]
        table[target] = rows
        have = rows.flatten()
        uses.index_add_(0, have.clamp(min=0).long(), (have >= 0).to(torch.int32))
        return s['k_cache'], s['v_cache'], table, uses
    for name in caches:
        s[name][s['target'].long()] = s[name][s['source'].long()]
    return s['k_cache'], s['v_cache']


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- in 64 bits, another way ------------------------------------------------------------------------------------

def _exact_attention(q, k, v, dout, window, sinks, scale):
    """Head by head over the whole matrix of scores, band by band of queries."""
    hq, sq, d = q.shape
    hk, sk, _ = k.shape
    outs, dqs = [], []
    dks, dvs = ([torch.zeros(sk, d, dtype=torch.float64, device=q.device) for _ in range(hk)] for _ in range(2))
    for h in range(hq):
        kd, vd = k[h * hk // hq].double(), v[h * hk // hq].double()
        o_h, dq_h = [], []
        for r0 in range(0, sq, 4096):
            qd = q[h, r0:r0 + 4096].double()
            age = (torch.arange(r0, r0 + len(qd), device=q.device) + sk - sq)[:, None] - torch.arange(sk, device=q.device)
            seen = (age >= 0) & (age < window)
            seen[:, :sinks] |= age[:, :sinks] >= 0
            e = torch.where(seen, qd @ kd.T * scale, -torch.inf)
            lse = torch.logsumexp(e, 1, keepdim=True)
            e = torch.where(seen, torch.exp(e - lse), 0.0)
            o = e @ vd
            o_h.append(o)
            if dout is None:
                continue
            do = dout[h, r0:r0 + 4096].double()
            dvs[h * hk // hq] += e.T @ do
            e *= do @ vd.T - (do * o).sum(1, keepdim=True)
            dq_h.append(e @ kd * scale)
            dks[h * hk // hq] += e.T @ qd * scale
        outs.append(torch.cat(o_h))
        if dout is not None:
            dqs.append(torch.cat(dq_h))
    out = torch.stack(outs)
    return out if dout is None else (out, torch.stack(dqs), torch.stack(dks), torch.stack(dvs))


def _exact_tree(s):
    c = s['case']
    q, page = s['q'], c['page']
    out = torch.empty(q.shape, dtype=torch.float64, device='cuda')
    table, lens = s['table'].tolist(), s['lengths'].tolist()
    parents = s['parents'].tolist() if s['parents'] is not None else [[-1]] * c['b']
    for b, n in enumerate(lens):
        end = n + c['t']
        order = torch.tensor(table[b][:-(-end // page)], device='cuda')
        k, v = (x[order].permute(1, 0, 2, 3).reshape(c['hk'], -1, c['d'])[:, :end].double().repeat_interleave(c['hq'] // c['hk'], 0)
                for x in (s['k_cache'], s['v_cache']))
        seen = torch.zeros(c['t'], end, dtype=torch.bool)
        for i in range(c['t']):
            chain = [i]
            while parents[b][chain[-1]] >= 0:
                chain.append(parents[b][chain[-1]])
            at = n + len(chain) - 1
            seen[i, :n] = True
            if c['window']:
                seen[i, min(c['sinks'], n):max(min(at - c['window'] + 1, n), min(c['sinks'], n))] = False
            for up, j in enumerate(chain):
                seen[i, n + j] = not c['window'] or up < c['window'] or at - up < c['sinks']
        e = torch.where(seen.to('cuda'), torch.bmm(q[b].double(), k.transpose(1, 2).contiguous()) * s['scale'], -torch.inf)
        out[b] = torch.bmm(torch.softmax(e, 2), v)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case['kind']
    if kind in ('step', 'prompt'):
        return _per_sequence(s, lambda q, k, v, dout=None: _exact_attention(q, k, v, dout, case['window'], case['sinks'], s['scale']))
    if kind == 'tree':
        return _exact_tree(s)
    if kind == 'copy':
        ways = dict(zip(s['target'].tolist(), s['source'].tolist()))
        order = torch.tensor([ways.get(p, p) for p in range(len(s['k_cache']))], device='cuda')
        return s['k_cache'].double()[order], s['v_cache'].double()[order]
    k, v = s['k_cache'].double(), s['v_cache'].double()
    if kind == 'append':
        lens, counts, path, table = (s[n].tolist() for n in ('lengths', 'counts', 'path', 'table'))
        for b, n in enumerate(lens):
            # a slot holds its drafted row, or the accepted one that moved there
            holds = [path[b][i] if i < counts[b] else i for i in range(case['t'])]
            for i, j in enumerate(holds):
                p, r = table[b][(n + i) // case['page']], (n + i) % case['page']
                k[p, :, r], v[p, :, r] = s['k'][b, :, j].double(), s['v'][b, :, j].double()
        return k, v, torch.tensor([n + m for n, m in zip(lens, counts)], dtype=torch.int32, device='cuda')
    for i in range(case['b'] if s['tail'] else 0):
        a, z = int(s['table'][i, s['full']]), int(s['spare'][i])
        k[z, :, :s['tail']], v[z, :, :s['tail']] = k[a, :, :s['tail']].clone(), v[a, :, :s['tail']].clone()
    return k, v, s['table'], s['uses']          # the losers hold the winners' pages already
