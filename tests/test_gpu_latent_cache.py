"""Attention over a cache of pages of latent rows, the pages of a batch's new rows, and the rows' way into them, against the 64-bit oracle and
plain Python: lengths around tiles, pages and pieces, one token and many, none, heads that fill no block, sequences that are not there, holes in the
page table, slots that hold anything.  Bounds: tests/_longctx.py."""
import math
import random

import pytest
import torch

from _longctx import assert_within, lse_bound, out_bound, score_error
from oracle import latent

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF, HF = torch.bfloat16, torch.float16


def _pool(lens, counts, E, page, dtype, seed, extra=5, columns=None, size=1.0):
    """cache with pages in any order, the table, lengths, starts; slots that belong to nobody hold NaN and inf"""
    g = torch.Generator().manual_seed(seed)
    ends = [max(n, 0) + m for n, m in zip(lens, counts)]
    need = [-(-n // page) for n in ends]
    columns = max(need) + 1 if columns is None else columns
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), columns), -1, dtype=torch.int32)
    rubbish = torch.tensor([float('nan'), float('inf')], dtype=dtype)
    cache = rubbish[torch.randint(0, 2, (pages, 1, page, E), generator=g)]
    at = 0
    for z, n in enumerate(ends):
        table[z, :need[z]] = torch.tensor(order[at:at + need[z]], dtype=torch.int32)
        at += need[z]
        for c in range(need[z]):
            m = min(page, n - c * page)
            cache[table[z, c], 0, :m] = (size * torch.randn(m, E, generator=g)).to(dtype)
    starts = torch.tensor([sum(counts[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    return cache, table, torch.tensor(lens, dtype=torch.int32), starts


def _run(q, cache, table, lens, starts, Ev, scale, max_length=None):
    from aotriton_amd import cache as ops
    return ops.latent_attention(*(t.to(DEV) for t in (q, cache, table, lens, starts)), Ev, scale, max_length, return_lse=True)


def _check(q, cache, table, lens, starts, Ev, scale, out, lse):
    want, want_lse, size = latent.cache_attention(q, cache, table, lens, starts, Ev, scale)
    clean = torch.where(torch.isfinite(cache.double()), cache.double(), 0.0)
    e = score_error(q, clean, scale)
    values = clean[..., :Ev].abs().amax() * (int(lens.max()) + int(starts[-1]) + 1) if lens.numel() else 0.0
    assert_within('out', out, want, out_bound(q.dtype, want, size, values, e))
    assert_within('lse', lse, want_lse, lse_bound(torch.where(want_lse.isinf(), 0.0, want_lse), e))


def _wide(table, page, room):
    """the table with `room` slots: how many rows a workgroup takes goes by that"""
    if not room:
        return table
    wide = torch.full((table.shape[0], room // page), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    return wide


CASES = [
    # lens, counts, Hq, E, Ev, page, dtype
    ([0], [1], 1, 576, 512, 16, BF),
    ([1], [1], 16, 576, 512, 16, HF),
    ([30, 31, 32, 33], [1, 1, 1, 1], 16, 576, 512, 16, BF),
    ([4095], [1], 16, 576, 512, 64, BF),
    ([4095], [1], 128, 576, 512, 64, HF),
    ([700, 3, 129], [1, 1, 1], 20, 576, 512, 32, HF),
    ([700, 3, 1200], [1, 1, 1], 64, 576, 512, 256, BF),
    ([500, 77, 0], [9, 1, 40], 7, 576, 512, 16, BF),
    ([100, 0, 64], [33, 0, 2], 128, 576, 512, 64, BF),
    ([0, 0], [65, 130], 4, 576, 512, 16, HF),
    ([333, 5], [3, 1], 32, 544, 512, 32, BF),
    ([333, 5], [3, 1], 32, 320, 256, 32, HF),
    ([97, 200], [4, 1], 5, 288, 256, 16, BF),
    ([97, 200], [4, 20], 16, 136, 128, 16, HF),
    ([97, 1], [1, 1], 3, 8, 8, 16, BF),
    ([97, 1], [1, 1], 3, 576, 8, 16, BF),
    ([300, 1], [1, 70], 9, 256, 256, 32, HF),
    ([300, 1], [1, 7], 40, 512, 512, 32, BF),
    ([300, 1], [1, 7], 40, 328, 264, 32, BF),
]


@pytest.mark.parametrize('lens,counts,Hq,E,Ev,page,dtype', CASES)
def test_latent_attention(lens, counts, Hq, E, Ev, page, dtype):
    cache, table, n, starts = _pool(lens, counts, E, page, dtype, seed=sum(lens) + E + Hq)
    q = torch.randn(sum(counts), Hq, E, generator=torch.Generator().manual_seed(1)).to(dtype)
    scale = 1.7 / math.sqrt(E)
    for top in (max(lens), 0, None):
        out, lse = _run(q, cache, table, n, starts, Ev, scale, top)
        _check(q, cache, table, n, starts, Ev, scale, out, lse)
    # a table with room for far more
    wide = torch.full((len(lens), (1 << 22) // page), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    out, lse = _run(q, cache, wide, n, starts, Ev, scale)
    _check(q, cache, table, n, starts, Ev, scale, out, lse)


@pytest.mark.parametrize('Hq,most', [(16, 1), (32, 1), (8, 20), (64, 3)])
def test_many_sequences(Hq, most):
    """more than a workgroup looks at in one go; some bring no token, some are not there"""
    rng = random.Random(Hq)
    lens = [rng.choice([0, 5, 40, 200, 333, -1]) for _ in range(600)]
    counts = [rng.choice([0, 1, 1, most]) for _ in lens]
    cache, table, n, starts = _pool(lens, counts, 136, 16, BF, seed=2)
    q = torch.randn(sum(counts), Hq, 136, generator=torch.Generator().manual_seed(3)).to(BF)
    out, lse = _run(q, cache, table, n, starts, 128, 0.1)
    _check(q, cache, table, n, starts, 128, 0.1, out, lse)


@pytest.mark.parametrize('Hq', [1, 3, 20, 32, 128])
@pytest.mark.parametrize('seed', [0, 1, 2])
def test_cuts_of_prompts_and_decoding(Hq, seed):
    """the list of work is cut anywhere: blocks of a prompt's rows that see one tile more from group to group, single tokens, sequences of a tile and
    less, one that takes most of the list; more rows of a block than a sequence has"""
    rng = random.Random(100 * seed + Hq)
    most = max(2, 1200 // Hq)
    lens = [rng.choice([0, rng.randint(1, 70), rng.randint(100, 900)]) for _ in range(6)] + [2500]
    counts = [rng.choice([1, 1, rng.randint(2, most), most]) for _ in range(6)] + [rng.choice([1, 40])]
    cache, table, n, starts = _pool(lens, counts, 576, rng.choice([16, 64]), HF, seed=seed)
    q = torch.randn(sum(counts), Hq, 576, generator=torch.Generator().manual_seed(seed)).half()
    out, lse = _run(q, cache, table, n, starts, 512, 0.05)
    _check(q, cache, table, n, starts, 512, 0.05, out, lse)


def test_rows_of_no_sequence():
    cache, table, n, starts = _pool([40, 70], [3, 2], 136, 16, HF, seed=4)
    q = torch.randn(11, 6, 136, generator=torch.Generator().manual_seed(5)).half()
    q[5:] = float('nan')
    out, lse = _run(q, cache, table, n, starts, 128, 0.1)
    _check(q[:5], cache, table, n, starts, 128, 0.1, out[:5], lse[:5])
    assert (out[5:] == 0).all() and torch.isposinf(lse[5:]).all()
    none = torch.zeros(0, dtype=torch.int32)
    out, lse = _run(q, cache, table[:0], none, torch.zeros(1, dtype=torch.int32), 128, 0.1)
    assert (out == 0).all() and torch.isposinf(lse).all()
    out, lse = _run(q[:0], cache, table, n, starts * 0, 128, 0.1)
    assert out.shape == (0, 6, 128) and lse.shape == (0, 6)


@pytest.mark.parametrize('E,Ev,room', [(320, 256, 0), (320, 256, 1 << 20), (576, 512, 0), (576, 512, 1 << 20)])
def test_holes_and_bad_indices(E, Ev, room):
    """pages outside the cache, lengths and offsets that name what is not there"""
    lens, counts = [500, 200, 90, 64], [2, 1, 3, 40]
    cache, table, n, starts = _pool(lens, counts, E, 16, BF, seed=6)
    table = _wide(table, 16, room)
    table[0, 3] = -1
    table[0, 7] = cache.shape[0]
    table[1, 0] = 2 ** 31 - 1
    table[1, 12] = -2 ** 31
    table[3] = -1                                     # nothing of it is there
    q = torch.randn(46, 16, E, generator=torch.Generator().manual_seed(7)).to(BF)
    out, lse = _run(q, cache, table, n, starts, Ev, 0.1)
    _check(q, cache, table, n, starts, Ev, 0.1, out, lse)
    assert (out[6:] == 0).all()

    def others(out2, lse2):
        """the sequences in front are what they were (the list of work is cut elsewhere then, and with a long table their sums are)"""
        assert room or torch.equal(out2[:3], out[:3])
        _check(q[:3], cache, table[:2], n[:2], starts[:3], Ev, 0.1, out2[:3], lse2[:3])
    n[2] = 2 ** 31 - 1                                # a length past the table: what the table has is seen
    others(*_run(q, cache, table, n, starts, Ev, 0.1))
    n[2] = -2 ** 31
    out2, lse2 = _run(q, cache, table, n, starts, Ev, 0.1)
    others(out2, lse2)
    assert (out2[3:6] == 0).all() and torch.isposinf(lse2[3:6]).all()
    wild = torch.tensor([-7, 2, 10 ** 9, 5, 46], dtype=torch.int32)
    n[2] = 90
    _run(q, cache, table, n, wild, Ev, 0.1)          # (whatever it gives, inside the tensors)
    out3, _ = _run(q, cache, table, n, starts, Ev, 0.1)
    assert torch.equal(out3, out)


@pytest.mark.parametrize('scale', [0.0, -0.05, 2.0])
@pytest.mark.parametrize('Hq', [16, 128])
@pytest.mark.parametrize('room', [0, 1 << 20])
def test_scales(room, scale, Hq):
    cache, table, n, starts = _pool([300, 20], [1, 2], 576, 16, BF, seed=8)
    table = _wide(table, 16, room)
    q = torch.randn(3, Hq, 576, generator=torch.Generator().manual_seed(9)).to(BF)
    out, lse = _run(q, cache, table, n, starts, 512, scale)
    _check(q, cache, table, n, starts, 512, scale, out, lse)


@pytest.mark.parametrize('order', [1, -1])
@pytest.mark.parametrize('Hq', [16, 64, 128])
@pytest.mark.parametrize('room', [0, 1 << 20])
def test_the_largest_scores_come_first_or_last(room, Hq, order):
    """the running maximum moves at every tile, or never"""
    cache, table, n, starts = _pool([900], [1], 576, 64, HF, seed=10)
    table = _wide(table, 64, room)
    size = torch.linspace(0.05, 4, 901)
    size = size if order > 0 else size.flip(0)
    for s in range(901):
        cache[table[0, s // 64], 0, s % 64] *= size[s].half()
    q = torch.randn(1, Hq, 576, generator=torch.Generator().manual_seed(11)).half()
    out, lse = _run(q, cache, table, n, starts, 512, 0.3)
    _check(q, cache, table, n, starts, 512, 0.3, out, lse)


def test_a_cache_beyond_31_bits():
    """pages whose rows lie past 2^31 elements, and 4 GiB, from the first"""
    page, E = 64, 576
    pages = (1 << 32) // (page * E * 2) + 3000
    cache = torch.empty(pages, 1, page, E, dtype=BF, device=DEV)
    small, table, n, starts = _pool([150, 70], [1, 1], E, page, BF, seed=12, extra=0)
    where = torch.arange(pages - small.shape[0], pages)
    cache[where.to(DEV)] = small.to(DEV)
    q = torch.randn(2, 16, E, generator=torch.Generator().manual_seed(13)).to(BF)
    far = torch.where(table >= 0, table + int(where[0]), -1)
    from aotriton_amd import cache as ops
    out, lse = ops.latent_attention(q.to(DEV), cache, far.to(torch.int32).to(DEV), n.to(DEV), starts.to(DEV), 512, 0.05, return_lse=True)
    _check(q, small, table, n, starts, 512, 0.05, out, lse)
    rows = torch.randn(2, 1, E, device=DEV).to(BF)
    slots = torch.tensor([(pages - 1) * page + 7, (pages - 2) * page], dtype=torch.int64, device=DEV)
    ops.append_packed(rows, None, cache, None, slots)
    assert torch.equal(cache[pages - 1, 0, 7], rows[0, 0]) and torch.equal(cache[pages - 2, 0, 0], rows[1, 0])


def test_strides():
    cache, table, n, starts = _pool([130, 40], [1, 5], 320, 16, HF, seed=14)
    q = torch.randn(6, 8, 320, generator=torch.Generator().manual_seed(15)).half()
    want = _run(q, cache, table, n, starts, 256, 0.1)
    from aotriton_amd import cache as ops
    ints = [t.to(DEV) for t in (table, n, starts)]
    wide = torch.full((cache.shape[0], 1, 16, 328), float('nan'), dtype=HF, device=DEV)
    wide[..., :320] = cache.to(DEV)
    heads_first = torch.empty(8, 6, 320, dtype=HF, device=DEV).transpose(0, 1).copy_(q)
    odd = torch.empty(q.numel() + 1, dtype=HF, device=DEV)[1:].view(q.shape).copy_(q)
    narrow = torch.full((2, table.shape[1] + 9), 5, dtype=torch.int32, device=DEV)[:, 4:4 + table.shape[1]].copy_(table)
    for qq, x, t in ((heads_first, wide[..., :320], ints[0]), (odd, cache.to(DEV), narrow)):
        got = ops.latent_attention(qq, x, t, *ints[1:], 256, 0.1, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_streams_and_schemas():
    from aotriton_amd import cache as ops
    cache, table, n, starts = (t.to(DEV) for t in _pool([2000, 30, 900], [1, 3, 1], 576, 64, BF, seed=16))
    q = torch.randn(5, 32, 576, device=DEV).to(BF)
    want = ops.latent_attention(q, cache, table, n, starts, 512, 0.05)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(ops.latent_attention(q, cache, table, n, starts, 512, 0.05))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)
    both = ('test_schema', 'test_faketensor')
    torch.library.opcheck(torch.ops.aotriton_amd.latent_cache_attention, (q, cache, table, n, starts, 512, 2000, 0.05), test_utils=both)
    slots = torch.tensor([3, -1, 70, 64, 9], dtype=torch.int64, device=DEV)
    rows = torch.randn(5, 1, 576, device=DEV).to(BF)
    torch.library.opcheck(torch.ops.aotriton_amd.cache_append_packed, (rows, None, cache, None, slots), test_utils=both)
    torch.library.opcheck(torch.ops.aotriton_amd.cache_append_packed, (rows, rows, cache, cache.clone(), slots), test_utils=both)
    torch.library.opcheck(torch.ops.aotriton_amd.cache_reserve, (table, torch.zeros(cache.shape[0], dtype=torch.int32, device=DEV), n, n * 0 + 1, 5, 64), test_utils=both)
    with pytest.raises(NotImplementedError, match='no gradient'):
        ops.latent_attention(q.requires_grad_(True), cache, table, n, starts, 512, 0.05)
    with pytest.raises(NotImplementedError, match='no gradient'):
        ops.append_packed(rows.requires_grad_(True), None, cache, None, slots)


# ---- reserve -------------------------------------------------------------------------------------------------------------

def _reserve(table, uses, lens, counts, tokens, slots):
    from aotriton_amd import cache as ops
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV).view(-1)
    t = torch.tensor(table, dtype=torch.int32, device=DEV).view(len(lens), len(table[0]) if table else 0)
    u = ints(uses)
    starts, slot_map, missing = ops.reserve(t, u, ints(lens), ints(counts), tokens, slots)
    assert slot_map.dtype == torch.int64 and starts.dtype == torch.int32 and missing.shape == (1,)
    want = latent.reserve(table, uses, lens, counts, tokens, slots)
    got = (t.tolist(), u.tolist(), starts.tolist(), slot_map.tolist(), int(missing))
    for name, a, b in zip(('table', 'uses', 'starts', 'slot map', 'missing'), got, want):
        assert a == b, name


@pytest.mark.parametrize('n,pages,columns,slots,top,most,room', [
    (1, 1, 1, 16, 0, 1, 1.0), (3, 40, 6, 16, 60, 30, 1.0), (7, 200, 12, 32, 200, 150, 1.0), (257, 5000, 9, 16, 100, 40, 1.0),
    (700, 300, 40, 64, 2000, 1, 1.0), (64, 70000, 600, 16, 5000, 4000, 1.0), (5, 64, 5, 256, 900, 300, 1.0), (20, 30, 8, 16, 60, 90, 1.0),
    (20, 400, 8, 16, 60, 60, 0.6), (2, 100000, 3000, 16, 30, 40000, 1.0)])
def test_reserve(n, pages, columns, slots, top, most, room):
    rng = random.Random(n + pages)
    lens = [rng.choice([0, rng.randint(0, top), rng.randint(0, top) // slots * slots]) for _ in range(n)]
    counts = [rng.choice([0, 1, 1, rng.randint(0, most), most]) for _ in range(n)]
    uses = [0] * pages
    table = [[-1] * columns for _ in range(n)]
    order = rng.sample(range(pages), pages)
    for z in range(n):
        for c in range(min(columns, -(-lens[z] // slots) + rng.choice([0, 0, 1]))):
            if order and rng.random() < 0.95:
                table[z][c] = order.pop()
                uses[table[z][c]] = rng.choice([1, 1, 2])
    _reserve(table, uses, lens, counts, int(sum(counts) * room), slots)
    _reserve(table, uses, lens, counts, sum(counts) + 13, slots)


def test_reserve_of_odd_calls():
    free = [0] * 9
    _reserve([[-1] * 4] * 4, [0] * 30, [-1, 5, 3, -2 ** 31], [4, -3, 20, 7], 24, 16)             # sequences that are not there, no rows
    _reserve([[-7, 99, 2 ** 31 - 1, 9]], free, [0], [64], 64, 16)                                # entries that name no page
    _reserve([[3, 1]], [1, 1, 0, 1, 0, 0, 1, 1, 1], [10], [40], 40, 16)                          # slots outside the table
    _reserve([[-1], [-1]], [5, -1, 3], [0, 0], [1, 1], 2, 16)                                    # no free page
    _reserve([[-1] * 3] * 2, free, [2 ** 31 - 1, 0], [5, 2 ** 31 - 1], 20, 16)                   # lengths and counts at the end of their type
    _reserve([[-1] * 3] * 3, free, [0, 0, 0], [2 ** 31 - 1] * 3, 33, 16)
    _reserve([[-1] * 3] * 2, free, [0, 0], [3, 4], 0, 16)                                        # no row
    _reserve([[], []], free, [0, 4], [3, 4], 9, 16)                                              # no column
    _reserve([[-1] * 3], [], [0], [3], 3, 16)                                                    # no page
    _reserve([], free, [], [], 3, 16)                                                            # no sequence


def test_reserve_of_a_large_pool():
    """more pages than have runs of 1024; free ones far behind"""
    pages, n = 5_000_000, 3
    uses = torch.ones(pages, dtype=torch.int32, device=DEV)
    free = torch.tensor([7, 63, 64, 1000, 4_000_000, 4_000_063, 4_999_998, 4_999_999], device=DEV)
    uses[free] = 0
    from aotriton_amd import cache as ops
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    table = torch.full((n, 4), -1, dtype=torch.int32, device=DEV)
    starts, slot_map, missing = ops.reserve(table, uses, ints(0, 0, 0), ints(40, 64, 33), 137, 16)
    assert table.tolist() == [[7, 63, 64, -1], [1000, 4_000_000, 4_000_063, 4_999_998], [4_999_999, -1, -1, -1]]
    assert int(missing) == 2 and starts.tolist() == [0, 40, 104, 137] and (uses == 1).all()
    assert slot_map[[0, 39, 40, 103, 104, 119, 120, 136]].tolist() == [112, 64 * 16 + 7, 16000, 4_999_998 * 16 + 15, 4_999_999 * 16, 4_999_999 * 16 + 15, -1, -1]


# ---- append_packed ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('rows,heads,E,Ev,page,slot_major,dtype', [
    (1, 1, 576, None, 16, False, BF), (300, 1, 320, None, 64, False, HF), (77, 8, 128, 128, 16, True, BF), (500, 3, 72, 40, 32, False, HF),
    (33, 2, 512, 64, 16, True, BF), (0, 1, 64, 64, 16, False, BF)])
def test_append_packed(rows, heads, E, Ev, page, slot_major, dtype):
    from aotriton_amd import cache as ops
    g = torch.Generator().manual_seed(rows)
    pages = rows // page + 4

    def cache(d):
        c = torch.randn(pages, page, heads, d, generator=g).to(dtype).transpose(1, 2)
        return c if slot_major else c.contiguous()
    caches = [cache(E)] + ([cache(Ev)] if Ev else [])
    new = [torch.randn(rows, heads, c.shape[3], generator=g).to(dtype) for c in caches]
    slots = torch.randperm(pages * page, generator=g)[:rows]
    if rows > 3:
        slots[torch.randperm(rows, generator=g)[:3]] = torch.tensor([-1, pages * page, 2 ** 62])
    mine = [c.to(DEV) for c in caches]
    dev = [t.to(DEV) for t in new]
    ops.append_packed(dev[0], dev[1] if Ev else None, mine[0], mine[1] if Ev else None, slots.to(DEV))
    for c, t, got in zip(caches, new, mine):
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                c[s // page, :, s % page] = t[i]
        assert torch.equal(got.cpu(), c)
    # rows that lie apart, or unaligned
    again = [c.to(DEV).clone() for c in caches]
    apart = [torch.zeros(rows, heads + 1, t.shape[2] + 4, dtype=dtype, device=DEV)[:, 1:, 4:].copy_(t) for t in new]
    ops.append_packed(apart[0], apart[1] if Ev else None, again[0], again[1] if Ev else None, slots.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(again, mine))


def test_writes_are_seen_by_autograd():
    from aotriton_amd import cache as ops
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    x = torch.zeros(4, 1, 16, 64, dtype=BF, device=DEV)
    v = x.clone()
    rows, slots = torch.ones(2, 1, 64, dtype=BF, device=DEV), torch.tensor([3, 20], device=DEV)
    table, uses = torch.full((1, 2), -1, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    for call, written in ((lambda: ops.append_packed(rows, rows, x, v, slots), (x, v)), (lambda: ops.append_packed(rows, None, x, None, slots), (x,)),
                          (lambda: ops.reserve(table, uses, ints(0), ints(1), 1, 16), (table, uses))):
        before = [t._version for t in written]
        call()
        assert [t._version for t in written] == [n + 1 for n in before]


# ---- together ----------------------------------------------------------------------------------------------------------------

def test_prompts_and_decoding_in_both_forms():
    """Latent vectors of a few sequences: a prompt in the expanded form; its latent rows into the cache; single tokens and chunks in the absorbed
    form, whose queries and results go through the projections that made keys and values.  Both say the same: every value against 64 bits, with what
    the roundings of the projected tensors leave."""
    from aotriton_amd import cache as ops, torch_ops
    H, L, R, E, Ev, page = 4, 256, 64, 64, 64, 16
    g = torch.Generator().manual_seed(30)
    rn = lambda *s: torch.randn(*s, generator=g)
    scale = 1 / math.sqrt(E + R)
    w_k, w_v = (rn(H, L, d) / math.sqrt(L) for d in (E, Ev))
    total = [150, 37, 200]
    rows = [torch.cat([rn(n, L), rn(n, R)], 1).to(BF) for n in total]           # latent vector and rotary part of every token
    qs = [rn(n, H, E + R).to(BF) for n in total]
    want = []
    for x, q in zip(rows, qs):
        c, r = x[:, :L].double(), x[:, L:].double()
        k, v = torch.einsum('nl,hle->hne', c, w_k.double()), torch.einsum('nl,hle->hne', c, w_v.double())
        want.append(latent.attention(q.double().transpose(0, 1), k, v, r, True, scale)[0].transpose(0, 1))
    pages, columns = 60, 14
    cache = torch.full((pages, 1, page, L + R), float('nan'), dtype=BF, device=DEV)
    table = torch.full((3, columns), -1, dtype=torch.int32, device=DEV)
    uses = torch.zeros(pages, dtype=torch.int32, device=DEV)
    lengths = torch.zeros(3, dtype=torch.int32, device=DEV)
    done = [0, 0, 0]
    # chunks of prompts next to single tokens
    for counts in ([100, 1, 64], [1, 20, 1], [1, 1, 100], [48, 0, 1], [0, 15, 34]):
        counts = [min(m, n - d) for m, n, d in zip(counts, total, done)]
        n = sum(counts)
        starts, slots, missing = ops.reserve(table, uses, lengths, torch.tensor(counts, dtype=torch.int32, device=DEV), n + 2, page)
        assert int(missing) == 0
        pick = [slice(d, d + m) for d, m in zip(done, counts)]
        new = torch.cat([x[p] for x, p in zip(rows, pick)] + [torch.zeros(2, L + R, dtype=BF)])
        q = torch.cat([t[p] for t, p in zip(qs, pick)] + [torch.zeros(2, H, E + R, dtype=BF)])
        ops.append_packed(new[:, None].to(DEV), None, cache, None, slots)
        absorbed = torch.cat([torch.einsum('nhe,hle->nhl', q[..., :E].float(), w_k), q[..., E:].float()], 2).to(BF)
        out = ops.latent_attention(absorbed.to(DEV), cache, table, lengths, starts, L, scale, max_length=200)
        got = torch.einsum('nhl,hle->nhe', out.cpu().double(), w_v.double())
        at = 0
        for z, p in enumerate(pick):
            # (the absorbed queries are rounded once, the result of the attention once: scores are off by a few steps, results with them)
            w = want[z][p]
            assert (got[at:at + counts[z]] - w).abs().max() < 0.05 if counts[z] else True
            at += counts[z]
        done = [d + m for d, m in zip(done, counts)]
        lengths += torch.tensor(counts, dtype=torch.int32, device=DEV)
    assert done == total and int((uses > 0).sum()) == sum(-(-n // page) for n in total)
    # the whole prompts at once, packed, in the expanded form
    x, q = torch.cat(rows), torch.cat(qs)
    k = torch.einsum('nl,hle->hne', x[:, :L].float(), w_k).to(BF)[None].to(DEV)
    v = torch.einsum('nl,hle->hne', x[:, :L].float(), w_v).to(BF)[None].to(DEV)
    cu = torch.tensor([0, 150, 187, 387], dtype=torch.int32, device=DEV)
    out = torch_ops.latent_attention(q.transpose(0, 1)[None].to(DEV), k, v, x[None, :, L:].to(DEV), scale=scale, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=200,
                                     max_seqlen_k=200)
    assert (out[0].transpose(0, 1).cpu().double() - torch.cat(want)).abs().max() < 0.05


def test_captured_serving_step():
    """reserve, append and attention in a graph, replayed with eager work between the replays"""
    from aotriton_amd import cache as ops
    E, Ev, page, tokens = 320, 256, 16, 12
    g = torch.Generator().manual_seed(40)
    start = torch.randn(40, 1, page, E, generator=g).to(BF).to(DEV)
    lens = torch.tensor([30, 0, 100], dtype=torch.int32, device=DEV)
    first = torch.full((3, 12), -1, dtype=torch.int32, device=DEV)
    first[0, :2] = torch.tensor([5, 9])
    first[2, :7] = torch.tensor([1, 2, 3, 30, 31, 33, 39])
    used = torch.zeros(40, dtype=torch.int32, device=DEV)
    used[torch.tensor([5, 9, 1, 2, 3, 30, 31, 33, 39], device=DEV)] = 1
    rows, q = torch.zeros(tokens, 1, E, dtype=BF, device=DEV), torch.zeros(tokens, 16, E, dtype=BF, device=DEV)
    counts = torch.tensor([1, 5, 1], dtype=torch.int32, device=DEV)

    def step(cache, table, uses, lens):
        starts, slots, missing = ops.reserve(table, uses, lens, counts, tokens, page)
        ops.append_packed(rows, None, cache, None, slots)
        out = ops.latent_attention(q, cache, table, lens, starts, Ev, 0.1, max_length=150)
        return out, starts, slots, missing
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step(start.clone(), first.clone(), used.clone(), lens)
    torch.cuda.current_stream().wait_stream(warm)
    mine, theirs = ([t.clone() for t in (start, first, used, lens)] for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*mine)
    for i in range(5):
        for t in (rows, q):
            t.copy_(torch.randn(t.shape, generator=g).to(BF))
        counts.copy_(torch.tensor([[1, 5, 1], [1, 1, 1], [0, 9, 3], [1, 1, 0], [4, 4, 4]][i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = step(*theirs)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(mine, theirs))
        for t in (mine[3], theirs[3]):
            t += counts


def test_compiled_serving_step():
    from aotriton_amd import cache as ops
    cache, table, n, starts = (t.to(DEV) for t in _pool([40, 7], [1, 1], 136, 16, BF, seed=50, extra=9))
    uses = torch.zeros(cache.shape[0], dtype=torch.int32, device=DEV)
    uses[table[table >= 0].long()] = 1
    rows, q, counts = torch.randn(4, 1, 136, device=DEV).to(BF), torch.randn(4, 6, 136, device=DEV).to(BF), torch.tensor([1, 3], dtype=torch.int32, device=DEV)

    def step(cache, table, uses, n):
        starts, slots, missing = ops.reserve(table, uses, n, counts, rows.shape[0], 16)
        ops.append_packed(rows, None, cache, None, slots)
        return ops.latent_attention(q, cache, table, n, starts, 128, 0.1).flatten(1), slots, missing
    torch._dynamo.reset()
    compiled = torch.compile(step, backend='aot_eager', fullgraph=True)
    a, b = ([t.clone() for t in (cache, table, uses, n)] for _ in range(2))
    for _ in range(2):
        assert all(torch.equal(x, y) for x, y in zip(step(*a), compiled(*b)))
        assert all(torch.equal(torch.nan_to_num(x), torch.nan_to_num(y)) for x, y in zip(a, b))


def test_forks_of_a_latent_cache():
    """the cache's other functions take it as two ranges of columns"""
    from aotriton_amd import cache as ops
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    cache, table, n, starts = (t.to(DEV) for t in _pool([40, 7], [0, 0], 576, 16, BF, seed=51, extra=6))
    uses = torch.zeros(cache.shape[0], dtype=torch.int32, device=DEV)
    uses[table[table >= 0].long()] = 1
    k, v = cache[..., :512], cache[..., 512:]
    ops.free(table, uses, ints(1), ints(0), ints(table.shape[1]))
    spare = (uses == 0).nonzero()[0].to(torch.int32)
    ops.fork(k, v, table, n, uses, ints(0), ints(1), spare)
    assert n.tolist() == [40, 40] and torch.equal(table[0, :2], table[1, :2]) and table[1, 2] == spare[0]
    assert torch.equal(cache[int(table[1, 2]), 0, :8], cache[int(table[0, 2]), 0, :8])
    rows = torch.randn(2, 1, 1, 576, device=DEV).to(BF)
    ops.append(rows[..., :512], rows[..., 512:], k, v, table, n)
    q = torch.randn(1, 16, 576, device=DEV).to(BF).expand(2, -1, -1)
    out = ops.latent_attention(q, cache, table, n, ints(0, 1, 2), 512, 0.05)
    assert not torch.equal(out[0], out[1])                       # their own last rows
    ops.append(rows[:1].expand(2, -1, -1, -1)[..., :512], rows[:1].expand(2, -1, -1, -1)[..., 512:], k, v, table, n)
    out = ops.latent_attention(q, cache, table, n, ints(0, 1, 2), 512, 0.05)
    assert torch.equal(out[0], out[1])


@pytest.mark.parametrize('Hq', [1, 16, 128])
@pytest.mark.parametrize('E,Ev,room', [(320, 256, 0), (320, 256, 1 << 18), (576, 512, 0), (576, 512, 1 << 18)])
def test_lengths_at_the_end_of_their_type(E, Ev, room, Hq):
    """past the table what the table has is seen, by all of a sequence's tokens, however far past it the length is: the results of a length that the
    table just holds"""
    lens, counts = [300, 90, 40], [2, 5, 1]
    cache, table, n, starts = _pool(lens, counts, E, 16, BF, seed=21)
    cache = torch.where(torch.isfinite(cache), cache, 0.25)
    narrow, table = table, _wide(table, 16, room)
    holds = table.shape[1] * 16
    q = torch.randn(8, Hq, E, generator=torch.Generator().manual_seed(22)).to(BF)
    n[1] = holds
    out, lse = _run(q, cache, table, n, starts, Ev, 0.1, 400)
    _check(q, cache, narrow, torch.clamp(n, max=narrow.shape[1] * 16), starts, Ev, 0.1, out, lse)
    for far in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 4, 2 ** 31 - 6, 2 ** 30):
        n[1] = far
        out2, lse2 = _run(q, cache, table, n, starts, Ev, 0.1, 400)
        assert torch.equal(out2, out) and torch.equal(lse2, lse), far
    for none in (-1, -2, -2 ** 31, -2 ** 31 + 3):
        n[1] = none
        out2, lse2 = _run(q, cache, table, n, starts, Ev, 0.1, 400)
        assert (out2[2:7] == 0).all() and torch.isposinf(lse2[2:7]).all()
