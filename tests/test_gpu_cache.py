"""The cache of pages and the attention of drafted tokens over it, against the 64-bit oracle: lengths around blocks, pages and parts, trees
with tokens that are not there, windows with sinks, holes in the page table, slots that hold anything.  Bounds: tests/_longctx.py."""
import ctypes
import math
import random

import pytest
import torch

from _longctx import assert_within, lse_bound, out_bound, score_error
from oracle import longctx

pytestmark = pytest.mark.gpu

DEV = 'cuda'


def _pool(lens, tokens, Hk, D, page, dtype, seed, Dv=None, extra=5, slot_major=True, columns=None):
    """caches with pages in any order, the table, and the lengths; slots that belong to nobody hold NaN and inf"""
    g = torch.Generator().manual_seed(seed)
    need = [-(-(max(n, 0) + tokens) // page) for n in lens]
    columns = max(need) + 1 if columns is None else columns
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), columns), -1, dtype=torch.int32)
    rubbish = torch.tensor([float('nan'), float('inf')], dtype=dtype)

    def cache(d):
        c = rubbish[torch.randint(0, 2, (pages, page, Hk, d), generator=g)]
        return c.transpose(1, 2) if slot_major else c.transpose(1, 2).contiguous()
    k, v = cache(D), cache(D if Dv is None else Dv)
    at = 0
    for z, n in enumerate(lens):
        table[z, :need[z]] = torch.tensor(order[at:at + need[z]], dtype=torch.int32)
        at += need[z]
        for s in range(max(n, 0) + tokens):
            for c in (k, v):
                c[table[z, s // page], :, s % page] = torch.randn(Hk, c.shape[3], generator=g).to(dtype)
    return k, v, table, torch.tensor(lens, dtype=torch.int32)


def _tree(rng, t, holes=0.0):
    return [-2 if rng.random() < holes else -1 if i == 0 or rng.random() < 0.15 else rng.randint(max(0, i - 4), i - 1) for i in range(t)]


def _run(q, k, v, table, lens, parents, window, sinks, scale, max_length=None):
    from aotriton_amd import cache
    dev = lambda t: None if t is None else t.to(DEV)
    return cache.tree_attention(dev(q), dev(k), dev(v), dev(table), dev(lens), dev(parents), max_length, window, sinks, scale, return_lse=True)


def _check(q, k, v, table, lens, parents, window, sinks, scale, out, lse):
    want, want_lse, size = longctx.tree_attention(q, k, v, table, lens, parents, window, sinks, scale)
    clean = lambda c: torch.where(torch.isfinite(c.double()), c.double(), 0.0)
    e = score_error(q, clean(k), scale)
    values = clean(v).abs().amax() * (int(lens.max()) + q.shape[2] + 1)
    assert_within('out', out, want, out_bound(q.dtype, want, size, values, e))
    assert_within('lse', lse, want_lse, lse_bound(torch.where(want_lse.isinf(), 0.0, want_lse), e))


CASES = [
    # lens, Hq, Hk, tokens, D, page, window, sinks, dtype, tree
    ([0], 1, 1, 1, 64, 16, 0, 0, torch.bfloat16, False),
    ([1], 4, 4, 1, 128, 16, 0, 0, torch.float16, False),
    ([31, 32, 33], 8, 2, 1, 128, 16, 0, 0, torch.bfloat16, False),
    ([15, 16, 17, 0], 4, 1, 2, 64, 16, 0, 0, torch.float16, True),
    ([4095], 32, 8, 1, 128, 64, 0, 0, torch.bfloat16, False),
    ([700, 3, 129], 8, 8, 1, 64, 32, 0, 0, torch.float16, False),
    ([500, 77], 8, 2, 9, 128, 16, 0, 0, torch.bfloat16, True),           # 36 packed rows
    ([100, 0, 64], 7, 1, 33, 64, 64, 0, 0, torch.bfloat16, True),
    ([1000, 40], 16, 2, 64, 128, 256, 0, 0, torch.float16, True),        # 512 rows
    ([300], 4, 4, 64, 64, 16, 0, 0, torch.float16, False),               # a chain
    ([900, 20, 333], 8, 2, 1, 128, 16, 100, 4, torch.bfloat16, False),
    ([900, 64, 5], 4, 2, 12, 64, 32, 64, 40, torch.float16, True),
    ([640, 700], 4, 1, 30, 128, 64, 5, 2, torch.bfloat16, False),        # a chain longer than the window
    ([640, 3], 4, 1, 40, 64, 16, 3, 5, torch.float16, True),
    ([200], 2, 2, 3, 64, 16, 1, 0, torch.bfloat16, False),               # nothing but itself
    ([50, 200], 2, 2, 3, 64, 16, 2000, 1000, torch.bfloat16, True),      # a window beyond everything
    ([333, 5], 6, 2, 5, 256, 32, 0, 0, torch.bfloat16, True),
    ([333, 5], 6, 2, 5, 200, 32, 77, 3, torch.float16, True),
    ([97], 3, 1, 4, 72, 16, 0, 0, torch.bfloat16, True),
    ([97, 1], 2, 1, 4, 40, 16, 0, 0, torch.float16, True),
]


@pytest.mark.parametrize('lens,Hq,Hk,tokens,D,page,window,sinks,dtype,tree', CASES)
def test_tree_attention(lens, Hq, Hk, tokens, D, page, window, sinks, dtype, tree):
    k, v, table, n = _pool(lens, tokens, Hk, D, page, dtype, seed=sum(lens) + D + tokens)
    g = torch.Generator().manual_seed(1)
    q = torch.randn(len(lens), tokens, Hq, D, generator=g).to(dtype).transpose(1, 2)
    rng = random.Random(tokens)
    parents = torch.tensor([_tree(rng, tokens) for _ in lens], dtype=torch.int32) if tree else None
    scale = 1 / math.sqrt(D)
    for top in (max(lens), 0, None):      # split for the lengths, hardly, and for the table's
        out, lse = _run(q, k, v, table, n, parents, window, sinks, scale, top)
        _check(q, k, v, table, n, parents, window, sinks, scale, out, lse)
    # a table for far more: what is planned for long caches has to do for these
    wide = torch.full((len(lens), (1 << 22) // page), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    out, lse = _run(q, k, v, wide, n, parents, window, sinks, scale)
    _check(q, k, v, table, n, parents, window, sinks, scale, out, lse)


@pytest.mark.parametrize('lens,Hq,Hk,tokens,D,page,window,sinks', [
    ([1000, 900], 64, 8, 64, 64, 16, 0, 0), ([1000, 63], 64, 8, 60, 128, 128, 500, 70), ([700, 650, 0, 5] * 4, 16, 8, 48, 64, 32, 0, 0),
    ([700, 128, 64, 1] * 4, 24, 8, 40, 120, 16, 600, 9)])
def test_tiles_of_short_caches(lens, Hq, Hk, tokens, D, page, window, sinks):
    k, v, table, n = _pool(lens, tokens, Hk, D, page, torch.float16, seed=40)
    table[0, 3] = -1
    rng = random.Random(41)
    parents = torch.tensor([_tree(rng, tokens, holes=0.1) for _ in lens], dtype=torch.int32)
    q = torch.randn(len(lens), tokens, Hq, D, generator=torch.Generator().manual_seed(42)).half().transpose(1, 2)
    out, lse = _run(q, k, v, table, n, parents, window, sinks, 1 / math.sqrt(D))
    pick = list(range(min(len(lens), 4)))
    _check(q[pick], k, v, table[pick], n[pick], parents[pick], window, sinks, 1 / math.sqrt(D), out[pick], lse[pick])


@pytest.mark.parametrize('lens,times,Hq,Hk,tokens,D,Dv,window,sinks', [
    ([1000, 63, 0], 1, 8, 2, 64, 256, 256, 0, 0), ([700, 129], 1, 16, 2, 40, 200, 136, 0, 0), ([600, 333], 1, 6, 1, 33, 136, 256, 100, 9),
    ([900, 5], 40, 8, 8, 64, 256, 256, 0, 0), ([1500, 0, 64], 30, 16, 4, 20, 192, 192, 300, 40), ([130, 1], 1, 32, 1, 2, 64, 160, 0, 0)])
def test_wide_heads_of_many_rows(lens, times, Hq, Hk, tokens, D, Dv, window, sinks):
    """head dims above 128: several blocks of 32 packed rows, in one piece and in several, in equal pieces of many sequences"""
    k, v, table, n = _pool(lens, tokens, Hk, D, 32, torch.bfloat16, seed=50, Dv=Dv)
    many = list(range(len(lens))) * times
    rng = random.Random(51)
    parents = torch.tensor([_tree(rng, tokens, holes=0.1) for _ in many], dtype=torch.int32)
    q = torch.randn(len(many), tokens, Hq, D, generator=torch.Generator().manual_seed(52)).bfloat16().transpose(1, 2)
    pick = sorted({0, 1, len(many) - 1})
    for top in (None, max(lens), 0):
        out, lse = _run(q, k, v, table[many], n[many], parents, window, sinks, 1 / math.sqrt(D), top)
        _check(q[pick], k, v, table[many][pick], n[many][pick], parents[pick], window, sinks, 1 / math.sqrt(D), out[pick], lse[pick])


def test_many_parts_of_a_long_cache():
    lens = [9000]
    k, v, table, n = _pool(lens, 1, 1, 64, 64, torch.bfloat16, seed=3)
    q = torch.randn(1, 4, 1, 64, generator=torch.Generator().manual_seed(2)).bfloat16()
    out, lse = _run(q, k, v, table, n, None, 0, 0, 0.125)
    _check(q, k, v, table, n, None, 0, 0, 0.125, out, lse)


@pytest.mark.parametrize('tokens,Hq,D,window', [(1, 8, 64, 0), (5, 16, 128, 0), (24, 32, 64, 0), (40, 64, 64, 0), (24, 32, 128, 1500)])
def test_equal_pieces_of_many_sequences(tokens, Hq, D, window):
    """more than 64 sequences, of very different lengths, cut into equal pieces: few rows, tiles of 128 and of 256"""
    rng = random.Random(tokens)
    lens = [rng.choice([0, 3, 60, 500, 1100, 1300]) for _ in range(69)] + [2900, 1, 1299]
    k, v, table, n = _pool(lens, tokens, 8, D, 64, torch.bfloat16, seed=30)
    q = torch.randn(len(lens), tokens, Hq, D, generator=torch.Generator().manual_seed(31)).bfloat16().transpose(1, 2)
    parents = torch.tensor([_tree(rng, tokens) for _ in lens], dtype=torch.int32)
    scale = 1 / math.sqrt(D)
    out, lse = _run(q, k, v, table, n, parents, window, 3 if window else 0, scale, 2900)
    pick = [0, 1, 2, 30, 62, 63, 64, 65, 69, 70, 71]
    _check(q[pick], k, v, table[pick], n[pick], parents[pick], window, 3 if window else 0, scale, out[pick], lse[pick])
    alone, alone_lse = _run(q, k, v, table, n, parents, window, 3 if window else 0, scale, 0)      # hardly split
    far = (alone.float() - out.float()).abs().amax((1, 2, 3))
    most = torch.where(torch.isfinite(v), v, 0.0).abs().max().item()
    assert (far <= 2 * 2.1 * 2.0 ** -8 * most).all()      # (two of out_bound's: 2.01 half steps of |V|, and what the scores are off by)


def _scratch(q, k, v, table, n, max_length):
    """fa_tree_attn through the C ABI: its result, and the bytes of scratch that it asks for"""
    from aotriton_amd._lib import fa_tree_params, lib
    from test_gpu_sinks import _view
    held, asked = [], []

    def alloc(_, size):
        asked.append(size)
        held.append(torch.empty(size, dtype=torch.uint8, device=DEV))
        return held[-1].data_ptr()

    class Allocator(ctypes.Structure):
        _fields_ = [('cookie', ctypes.c_void_p), ('alloc', ctypes.CFUNCTYPE(ctypes.c_void_p, ctypes.c_void_p, ctypes.c_uint64))]
    a = Allocator()
    a.alloc = Allocator._fields_[1][1](alloc)
    p = fa_tree_params()
    out = torch.empty_like(q)
    for view, t in ((p.Q, q), (p.Out, out), (p.cache.K, k), (p.cache.V, v), (p.cache.table, table), (p.cache.lengths, n)):
        _view(view, t)
    p.Sm_scale, p.max_length = 0.125, max_length
    assert lib.fa_tree_attn(ctypes.byref(p), torch.cuda.current_stream().cuda_stream, ctypes.byref(a)) == 0
    torch.cuda.synchronize()
    return out, sum(asked)


@pytest.mark.parametrize('B,tokens,length,columns', [(8, 64, 4096, 2048), (1, 1, 2048, 4096), (8, 1, 300, 8192)])
def test_scratch_follows_the_lengths(B, tokens, length, columns):
    """a table for much longer sequences changes neither how the keys are cut nor the scratch"""
    page, Hq, Hk, D = 64, 32, 8, 128
    need = -(-(length + tokens) // page)
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(need * 2, Hk, page, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    table = torch.full((B, columns), -1, dtype=torch.int32, device=DEV)
    table[:, :need] = torch.randint(0, need * 2, (B, need), device=DEV, generator=g, dtype=torch.int32)
    n = torch.full((B,), length, dtype=torch.int32, device=DEV)
    q = torch.randn(B, Hq, tokens, D, device=DEV, generator=g).bfloat16()
    out, narrow = _scratch(q, k, v, table[:, :need].contiguous(), n, length)
    far, wide = _scratch(q, k, v, table, n, length)
    assert torch.equal(out, far)
    assert narrow == wide


def test_scratch_of_many_sequences():
    """the sums of sequences that lie in several pieces are of a number that the chip sets, not the sequences"""
    page, tokens, Hq, Hk, D, length = 64, 64, 8, 2, 64, 2000
    need = -(-(length + tokens) // page)
    g = torch.Generator(device=DEV).manual_seed(2)
    k, v = (torch.randn(need, Hk, page, D, device=DEV, generator=g).half() for _ in range(2))
    asked = []
    for B in (300, 600):
        table = torch.arange(need, dtype=torch.int32, device=DEV).expand(B, need).contiguous()
        n = torch.full((B,), length, dtype=torch.int32, device=DEV)
        q = torch.randn(B, Hq, tokens, D, device=DEV, generator=g).half()
        out, size = _scratch(q, k, v, table, n, length)
        asked.append(size)
    assert asked[0] == asked[1] <= 128 << 20


@pytest.mark.parametrize('lens,times,tokens,Hq,D,top,window', [
    ([3000, 500, 0], 1, 1, 8, 64, 700, 0), ([3000, 500, 0], 1, 6, 8, 128, 700, 0), ([2500, 64], 12, 40, 16, 128, 900, 0), ([2500, 64], 20, 24, 8, 64, 600, 0),
    ([1200, 3], 2, 4, 8, 256, 300, 0), ([1500, 3], 1, 2, 8, 64, 900, 800)])
def test_sequences_longer_than_planned(lens, times, tokens, Hq, D, top, window):
    """the last piece of a sequence has what is left of it"""
    k, v, table, n = _pool(lens, tokens, 2, D, 16, torch.float16, seed=85)
    many = list(range(len(lens))) * times
    rng = random.Random(86)
    parents = torch.tensor([_tree(rng, tokens) for _ in many], dtype=torch.int32)
    q = torch.randn(len(many), tokens, Hq, D, generator=torch.Generator().manual_seed(87)).half().transpose(1, 2)
    out, lse = _run(q, k, v, table[many], n[many], parents, window, 3 if window else 0, 1 / math.sqrt(D), top)
    pick = sorted({0, 1, len(many) - 2, len(many) - 1})
    _check(q[pick], k, v, table[many][pick], n[many][pick], parents[pick], window, 3 if window else 0, 1 / math.sqrt(D), out[pick], lse[pick])


@pytest.mark.parametrize('tokens,Hq', [(1, 2), (20, 8)])
def test_a_visible_nan_stays(tokens, Hq):
    k, v, table, n = _pool([300, 40], tokens, 2, 64, 16, torch.float16, seed=32)
    k[table[0, 3], 0, 5] = float('nan')
    v[table[1, 1], 1, 2] = float('nan')
    q = torch.randn(2, Hq, tokens, 64, generator=torch.Generator().manual_seed(33)).half()
    for top in (None, 0):
        out, _ = _run(q, k, v, table, n, None, 0, 0, 0.125, top)
        half = Hq // 2
        assert out[0, :half].isnan().all() and out[1, half:].isnan().all()
        assert torch.isfinite(out[0, half:]).all() and torch.isfinite(out[1, :half]).all()


@pytest.mark.parametrize('window', [0, 20])
def test_tokens_that_are_not_there(window):
    lens, tokens = [70, 33, 0], 21
    k, v, table, n = _pool(lens, tokens, 2, 64, 16, torch.float16, seed=4)
    rng = random.Random(5)
    rows = [_tree(rng, tokens, holes=0.25) for _ in lens]
    rows[0][3], rows[0][7], rows[1][0] = 3, 9, 5            # itself, a later one, a later one
    rows[2] = [-2] * tokens                                 # nothing at all
    parents = torch.tensor(rows, dtype=torch.int32)
    # what is not there may hold anything
    for z in range(3):
        for t in range(tokens):
            if longctx.chain(rows[z], t) is None:
                s = lens[z] + t
                k[table[z, s // 16], :, s % 16] = float('inf')
                v[table[z, s // 16], :, s % 16] = float('nan')
    q = torch.randn(3, 4, tokens, 64, generator=torch.Generator().manual_seed(6)).half()
    wide = torch.full((3, 1 << 18), -1, dtype=torch.int32)      # (of 16 slots: planned for a long cache)
    wide[:, :table.shape[1]] = table
    for t in (wide, table):
        out, lse = _run(q, k, v, t, n, parents, window, 2 if window else 0, 0.125)
        _check(q, k, v, table, n, parents, window, 2 if window else 0, 0.125, out, lse)
    assert (out[2] == 0).all() and torch.isinf(lse[2]).all()


@pytest.mark.parametrize('lens,tokens,Hq,Hk,D', [([700, 140, 40], 5, 4, 2, 64), ([900, 300], 12, 8, 2, 128), ([600, 200], 40, 16, 2, 64), ([300, 5], 4, 2, 2, 256)])
def test_queries_of_tokens_that_are_not_there(lens, tokens, Hq, Hk, D):
    """they may be anything: scores that overflow to inf or are NaN, in slots that every other token sees whole"""
    k, v, table, n = _pool(lens, tokens, Hk, D, 16, torch.bfloat16, seed=70)
    rng = random.Random(71)
    rows = [_tree(rng, tokens, holes=0.3) for _ in lens]
    rows[0][1], rows[0][2] = -2, -1
    gone = torch.tensor([[longctx.chain(r, t) is None for t in range(tokens)] for r in rows])
    parents = torch.tensor(rows, dtype=torch.int32)
    clean = torch.randn(len(lens), Hq, tokens, D, generator=torch.Generator().manual_seed(72)).bfloat16()
    clean[gone[:, None].expand(-1, Hq, -1)] = 0
    for value, columns in ((3e38, 1), (3e38, D), (math.inf, 1), (-math.inf, 1), (math.inf, D), (math.nan, D)):
        q = clean.clone()
        q[..., :columns][gone[:, None, :].expand(-1, Hq, -1)] = value
        for top in (None, max(lens), 0):
            out, lse = _run(q, k, v, table, n, parents, 0, 0, 1 / math.sqrt(D), top)
            _check(clean, k, v, table, n, parents, 0, 0, 1 / math.sqrt(D), out, lse)
            many = list(range(len(lens))) * 48                 # (equal pieces)
            far, far_lse = _run(q[many], k, v, table[many], n[many], parents[many], 0, 0, 1 / math.sqrt(D), top)
            _check(clean, k, v, table, n, parents, 0, 0, 1 / math.sqrt(D), far[-len(lens):], far_lse[-len(lens):])


def test_bad_lengths_and_pages():
    """a negative length, lengths past the table, entries that are no pages: what they stand for is not there"""
    lens, tokens, page = [100, 200, 60, 150], 3, 16
    k, v, table, n = _pool(lens, tokens, 2, 64, page, torch.bfloat16, seed=7)
    k, v = (torch.where(torch.isfinite(c.float()), c, torch.zeros_like(c)) for c in (k, v))
    n[0] = -5
    n[1] = table.shape[1] * page - 1                         # the drafted tokens lie behind the table's end, all but one
    table[2, 1] = k.shape[0]
    table[2, 2] = 2 ** 31 - 1
    table[3, :3] = -(2 ** 31)
    table[1, 5] = -1
    q = torch.randn(4, 4, tokens, 64, generator=torch.Generator().manual_seed(8)).bfloat16()
    parents = torch.tensor([[-1, 0, 0]] * 4, dtype=torch.int32)
    for window, sinks in ((0, 0), (50, 20)):
        out, lse = _run(q, k, v, table, n, parents, window, sinks, 0.125)
        _check(q, k, v, table, n, parents, window, sinks, 0.125, out, lse)
        many = [0, 1, 2, 3] * 64                             # (enough of them for tiles)
        far, far_lse = _run(q[many], k, v, table[many], n[many], parents[many], window, sinks, 0.125)
        _check(q[:4], k, v, table, n, parents, window, sinks, 0.125, far[:4], far_lse[:4])
        assert all(torch.equal(far[i:i + 4], far[:4]) for i in range(0, 256, 4))
    assert (out[0] == 0).all()


@pytest.mark.parametrize('past', [1, 10, 100, 2 ** 31 - 1])
@pytest.mark.parametrize('tokens,Hq', [(1, 4), (3, 4), (40, 16)])
def test_a_window_behind_the_table(past, tokens, Hq):
    """of a sequence that is longer than its row of the table the sinks are still there"""
    page, columns, window, sinks = 16, 6, 10, 20
    room = page * columns
    k, v, table, _ = _pool([room], 0, 2, 64, page, torch.bfloat16, seed=73, columns=columns)
    table = table.expand(3, columns).clone()
    table[1, 1] = -1
    n = torch.tensor([min(room + past, 2 ** 31 - 1), min(room + past, 2 ** 31 - 2), room], dtype=torch.int64).int()
    q = torch.randn(3, Hq, tokens, 64, generator=torch.Generator().manual_seed(74)).bfloat16()
    # (the oracle goes through all slots: a length that the window leaves the table behind by)
    same = torch.tensor([min(room + past, 3 * room), min(room + past, 3 * room), room], dtype=torch.int32)
    for w, s in ((window, sinks), (1, 1), (window, 5000), (1, 0)):
        out, lse = _run(q, k, v, table, n, None, w, s, 0.125)
        _check(q, k, v, table, same, None, w, s, 0.125, out, lse)
        many = [0, 1, 2] * 80
        far, far_lse = _run(q[many], k, v, table[many], n[many], None, w, s, 0.125)
        _check(q, k, v, table, same, None, w, s, 0.125, far[-3:], far_lse[-3:])


def test_released_pages_under_a_window():
    """pages between the sinks and the window go back to the pool and are somebody else's"""
    from aotriton_amd import cache
    lens, page, window, sinks = [600, 310], 16, 64, 4
    k, v, table, n = _pool(lens, 1, 2, 64, page, torch.float16, seed=9)
    q = torch.randn(2, 4, 1, 64, generator=torch.Generator().manual_seed(10)).half()
    k, v, table, n, q = (t.to(DEV) for t in (k, v, table, n, q))
    want = cache.tree_attention(q, k, v, table, n, window=window, sinks=sinks)
    uses = torch.zeros(k.shape[0], dtype=torch.int32, device=DEV)
    uses[table[table >= 0].long()] = 1
    before = table.clone()
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    cache.free(table, uses, ints(0, 1), ints(1, 1), (n - window + 1) // page)
    gone = before[(before >= 0) & (table < 0)].long()
    assert len(gone) == (600 - 63) // 16 - 1 + (310 - 63) // 16 - 1 and (uses[gone] == 0).all()
    k[gone], v[gone] = float('nan'), float('nan')
    assert torch.equal(cache.tree_attention(q, k, v, table, n, window=window, sinks=sinks), want)


def test_value_head_dim_heads_first_and_strides():
    lens, tokens = [130, 64], 4
    k, v, table, n = _pool(lens, tokens, 2, 64, 32, torch.bfloat16, seed=11, Dv=128, slot_major=False)
    q = torch.randn(2, 6, tokens, 64, generator=torch.Generator().manual_seed(12)).bfloat16()
    wide = torch.zeros(2, 9, dtype=torch.int32)[:, 2:2 + table.shape[1]].copy_(table)      # rows of a bigger table
    out, lse = _run(q, k, v, table, n, None, 0, 0, 0.125)
    _check(q, k, v, table, n, None, 0, 0, 0.125, out, lse)
    out2, _ = _run(q, k, v, wide, n, None, 0, 0, 0.125)
    assert torch.equal(out, out2)
    odd = torch.empty(2, 6, tokens, 67, dtype=q.dtype)[..., 1:65].copy_(q)
    assert torch.equal(_run(odd, k, v, table, n, None, 0, 0, 0.125)[0], out)


@pytest.mark.parametrize('scale', [0.0, -0.3, 8.0])
def test_scales(scale):
    k, v, table, n = _pool([90], 2, 1, 64, 16, torch.bfloat16, seed=13)
    q = torch.randn(1, 2, 2, 64, generator=torch.Generator().manual_seed(14)).bfloat16()
    out, lse = _run(q, k, v, table, n, None, 0, 0, scale)
    _check(q, k, v, table, n, None, 0, 0, scale, out, lse)


# ---- rows, pages and sequences: everything is exact ---------------------------------------------------------------

def _equal(a, b):
    as_int = lambda t: t.cpu().contiguous().view(torch.int16)
    assert torch.equal(as_int(a), as_int(b))


@pytest.mark.parametrize('page,Hk,D,Dv,slot_major', [(16, 1, 64, 64, True), (64, 8, 128, 128, True), (32, 3, 72, 40, False)])
def test_append_and_keep(page, Hk, D, Dv, slot_major):
    from aotriton_amd import cache
    lens, tokens, steps = [0, 15, 16, 100, -3, 47], 20, 9
    k, v, table, n = _pool(lens, tokens, Hk, D, page, torch.float16, seed=15, Dv=Dv, slot_major=slot_major)
    table[3, (100 + 5) // page] = -1                             # a hole: what goes there is dropped
    g = torch.Generator().manual_seed(16)
    nk = torch.randn(6, tokens, Hk, D, generator=g).half().transpose(1, 2)
    nv = torch.randn(6, tokens, Hk, Dv, generator=g).half().transpose(1, 2)
    counts = torch.tensor([20, 7, 0, 20, 20, 25], dtype=torch.int32)
    rng = random.Random(17)
    path = torch.tensor([sorted(rng.sample(range(tokens), steps)) for _ in lens], dtype=torch.int32)
    kept = torch.tensor([9, 4, 0, 9, 3, 30], dtype=torch.int32)
    dk, dv, dt, dn = (t.to(DEV) for t in (k, v, table, n))
    cache.append(nk.to(DEV), nv.to(DEV), dk, dv, dt, dn, counts.to(DEV))
    where = lambda z, s: (int(table[z, s // page]), s % page) if s // page < table.shape[1] and table[z, s // page] >= 0 else None
    for z in range(6):
        for t in range(min(tokens, int(counts[z]))):
            at = where(z, lens[z] + t) if lens[z] >= 0 else None
            if at:
                k[at[0], :, at[1]], v[at[0], :, at[1]] = nk[z, :, t], nv[z, :, t]
    _equal(dk, k)
    _equal(dv, v)
    after = cache.keep_path(dk, dv, dt, dn, path.to(DEV), kept.to(DEV))
    for z in range(6):
        if lens[z] < 0:
            continue
        for i in range(min(int(kept[z]), steps)):
            a, b = where(z, lens[z] + int(path[z, i])), where(z, lens[z] + i)
            if a and b:
                k[b[0], :, b[1]], v[b[0], :, b[1]] = k[a[0], :, a[1]].clone(), v[a[0], :, a[1]].clone()
    _equal(dk, k)
    _equal(dv, v)
    assert after.tolist() == [9, 19, 16, 109, -3, 56]
    assert dn.tolist() == lens


@pytest.mark.parametrize('layout', ['slots first', 'heads first', 'apart'])
def test_copy_pages(layout):
    from aotriton_amd import cache
    g = torch.Generator().manual_seed(18)
    k, v = torch.randn(12, 16, 3, 72, generator=g).bfloat16(), torch.randn(12, 16, 3, 72, generator=g).bfloat16()
    if layout == 'heads first':
        k, v = k.view(12, 3, 16, 72), v.view(12, 3, 16, 72)
        dk, dv = k.to(DEV), v.to(DEV)
    else:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
        dk, dv = (t.to(DEV) for t in (k, v))
        if layout == 'apart':
            dk = torch.zeros(12, 3, 20, 80, dtype=k.dtype, device=DEV)[:, :, :16, :72].copy_(k)
    source, target = [0, 5, 5, -1, 12, 7, 2], [3, 1, 9, 4, 6, 7, 40]
    cache.copy_pages(dk, dv, *(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (source, target)))
    for a, b in ((0, 3), (5, 1), (5, 9)):
        k[b], v[b] = k[a].clone(), v[a].clone()
    _equal(dk, k)
    _equal(dv, v)


def test_fork_and_free():
    from aotriton_amd import cache
    page, lens = 16, [40, 32, 7, 0, 16]
    k, v, table, n = _pool(lens + [0] * 5, 0, 2, 64, page, torch.float16, seed=19, extra=8, columns=300)
    pages = k.shape[0]
    table[0, 1] = -1                                             # a released page
    used = set(table[table >= 0].tolist())
    unused = [p for p in range(pages) if p not in used]
    uses = torch.zeros(pages, dtype=torch.int32)
    uses[table[table >= 0].long()] = 1
    table[9, :4] = torch.tensor([3, 4, 5, 6], dtype=torch.int32)    # overwritten
    source, target = [0, 0, 1, 2, 3, 4, 99], [5, 6, 7, 8, 9, -1, 3]
    spare = unused[:2] + [pages + 1] + unused[2:3] + [-1, 0, 0]
    dk, dv, dt, dn, du = (t.to(DEV) for t in (k, v, table, n, uses))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    cache.fork(dk, dv, dt, dn, du, ints(source), ints(target), ints(spare))
    for a, b, x in list(zip(source, target, spare))[:5]:
        full, tail = divmod(lens[a], page)
        row = table[a].clone()
        row[full:] = -1
        if tail:
            k[x, :, :tail], v[x, :, :tail] = k[table[a, full], :, :tail], v[table[a, full], :, :tail]
            row[full] = x
        table[b] = row
        n[b] = lens[a]
        for p in row[row >= 0].tolist():
            uses[p] += 1
    _equal(dk, k)
    _equal(dv, v)
    assert torch.equal(dt.cpu(), table) and torch.equal(dn.cpu(), n) and torch.equal(du.cpu(), uses)
    # the first sequence goes, twice in one call; another one's first page; nothing; a sequence that is not there
    cache.free(dt, du, ints([0, 0, 7, 1, 50, -1]), ints([0, 0, 0, 5, 0, 0]), ints([300, 1000, 1, 2, 9, 9]))
    for p in table[0][table[0] >= 0].tolist() + [int(table[7, 0])]:
        uses[p] -= 1
    table[0] = -1
    table[7, 0] = -1
    assert torch.equal(dt.cpu(), table) and torch.equal(du.cpu(), uses)


def test_a_fork_of_rows_that_are_not_there():
    """the partial page of the source is no page: the spare one stays free"""
    from aotriton_amd import cache
    page = 16
    k, v, table, n = _pool([40, 24, 20, 7, 5], 0, 2, 64, page, torch.float16, seed=75, extra=8, columns=4)
    table = torch.cat([table, torch.tensor([[0, 1, 2, 3]] * 5, dtype=torch.int32)])
    n = torch.cat([n, torch.full((5,), 9, dtype=torch.int32)])
    table[0, 2], table[1, 1], table[2, 1] = -1, k.shape[0], -(2 ** 31)
    used = set(table[:5].flatten().tolist())
    spare = [p for p in range(k.shape[0]) if p not in used][:5]
    uses = torch.zeros(k.shape[0], dtype=torch.int32)
    dk, dv, dt, dn, du = (t.to(DEV) for t in (k, v, table, n, uses))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    cache.fork(dk, dv, dt, dn, du, ints([0, 1, 2, 3, 4]), ints([5, 6, 7, 8, 9]), ints(spare))
    want, want_n = table.clone(), n.clone()
    for a, b in ((0, 5), (1, 6), (2, 7), (3, 8), (4, 9)):
        full = int(n[a]) // page
        want[b] = -1
        want[b, :full] = table[a, :full]
        want_n[b] = n[a]
        for p in table[a, :full].tolist():
            uses[p] += 1
    for a, b, rows in ((3, 8, 7), (4, 9, 5)):
        want[b, 0] = spare[a]
        uses[spare[a]] += 1
        k[spare[a], :, :rows], v[spare[a], :, :rows] = k[table[a, 0], :, :rows].clone(), v[table[a, 0], :, :rows].clone()
    assert torch.equal(dt.cpu(), want)
    assert torch.equal(dn.cpu(), want_n) and torch.equal(du.cpu(), uses)
    _equal(dk, k)
    _equal(dv, v)


def test_a_sequence_that_is_not_there_has_no_fork():
    from aotriton_amd import cache
    k, v, table, n = _pool([40, 24, 20, 7], 0, 2, 64, 16, torch.float16, seed=76, extra=3)
    n[0], n[1] = -1, -(2 ** 31)
    uses = torch.zeros(k.shape[0], dtype=torch.int32)
    dk, dv, dt, dn, du = (t.to(DEV) for t in (k, v, table, n, uses))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    cache.fork(dk, dv, dt, dn, du, ints(0, 1), ints(2, 3), ints(8, 9))
    assert torch.equal(dt.cpu(), table) and torch.equal(dn.cpu(), n) and torch.equal(du.cpu(), uses)
    _equal(dk, k)
    _equal(dv, v)


def test_a_fork_without_columns():
    from aotriton_amd import cache
    k, v, _, _ = (t.to(DEV) for t in _pool([40], 0, 2, 64, 16, torch.float16, seed=77))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    lengths, uses = ints(0, 7, 9), torch.zeros(k.shape[0], dtype=torch.int32, device=DEV)
    cache.fork(k, v, torch.empty(3, 0, dtype=torch.int32, device=DEV), lengths, uses, ints(1), ints(0), ints(2))
    assert lengths.tolist() == [7, 7, 9] and (uses == 0).all()


@pytest.mark.parametrize('window,sinks', [(0, 0), (90, 4)])
def test_a_prompt_then_drafted_tokens(window, sinks):
    """The operators together: a prompt goes through attention with sinks into the cache, the sequence is forked, trees are drafted,
    attended and kept, and what the tokens get equals attention over the whole sequence at once."""
    from aotriton_amd import cache, torch_ops
    B, Hq, Hk, D, page, prompt, tokens, dt = 2, 4, 2, 64, 16, 75, 6, torch.bfloat16
    g = torch.Generator().manual_seed(21)
    rn = lambda h, n: torch.randn(B, n, h, D, generator=g).to(dt).to(DEV).transpose(1, 2)
    total = prompt + 2 * tokens
    w = window or 10 ** 6
    qs, ks, vs = rn(Hq, prompt), rn(Hk, prompt), rn(Hk, prompt)
    columns = -(-total // page) + 1
    k = torch.full((60, page, Hk, D), float('nan'), dtype=dt, device=DEV).transpose(1, 2)
    v = k.clone()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    table = ints([list(range(z * columns, (z + 1) * columns)) for z in range(B)] + [[-1] * columns] * B)
    uses = torch.zeros(60, dtype=torch.int32, device=DEV)
    uses[:B * columns] = 1
    lengths = ints([0] * B)
    for at in range(0, prompt, 50):
        cache.append(ks[:, :, at:at + 50], vs[:, :, at:at + 50], k, v, table[:B], lengths + at)
    lengths = ints([prompt] * B + [0] * B)
    cache.fork(k, v, table, lengths, uses, ints([0, 1]), ints([2, 3]), ints([50, 51]))
    table[2:, prompt // page + 1:prompt // page + 2] = ints([[52], [53]])      # room for the drafts
    assert lengths.tolist() == [prompt] * 4
    grow = [(ks, vs, qs)]
    for step in range(2):
        q, nk, nv = rn(Hq, tokens), rn(Hk, tokens), rn(Hk, tokens)
        parents = ints([[-1, 0, 0, 1, 2, 3], [-1, 0, 1, 1, -1, 4]])
        path, counts = ints([[0, 1, 3, 5], [0, 1, 3, 3]]), ints([4, 3])
        both = lambda t: torch.cat([t, t])
        cache.append(both(nk), both(nv), k, v, table, lengths)
        out = cache.tree_attention(both(q), k, v, table, lengths, both(parents), window=window, sinks=sinks)
        assert torch.equal(out[:B], out[B:])                               # the fork sees what its source sees
        after = cache.keep_path(k, v, table, lengths, both(path), both(counts))
        if step == 0:
            # the accepted path as a sequence of its own, all at once
            for z in range(B):
                take = path[z, :counts[z]].long()
                kk, vv, qq = (torch.cat([a[z], b[z][:, take]], 1)[None] for a, b in ((ks, nk), (vs, nv), (qs, q)))
                whole = torch_ops.sink_attention(qq, kk, vv, w, sinks)[0, :, prompt:]
                seen = longctx.sink_mask(qq.shape[2], kk.shape[2], w, sinks)
                want, _, p = longctx.attention(qq[0].cpu(), kk[0].cpu(), vv[0].cpu(), seen, D ** -0.5)
                size = torch.matmul(p, vv[0].cpu().double().abs().repeat_interleave(2, 0))
                bound = out_bound(dt, want, size, vv.abs().sum().cpu().double(), score_error(qq, kk, D ** -0.5))[:, prompt:]
                assert_within('tree', out[z][:, take], want[:, prompt:], bound)
                assert_within('whole', whole, want[:, prompt:], bound)
                rows, there = longctx.rows_of(k.cpu(), table[z].tolist(), int(after[z]))
                assert there.all()
                _equal(rows, kk[0])
        lengths = after
    assert lengths.tolist() == [prompt + 8, prompt + 6] * 2
    cache.free(table, uses, ints([0, 1, 2, 3]), ints([0] * 4), ints([columns] * 4))
    assert (table == -1).all()
    assert (uses[:B * columns] == 0).all() and (uses[50:52] == 0).all()


def test_captured_serving_step():
    """append, attention and keep in a graph, replayed with eager work between the replays"""
    from aotriton_amd import cache
    lens, tokens = [300, 45], 8
    k, v, table, n = (t.to(DEV) for t in _pool(lens, tokens * 4, 2, 64, 16, torch.bfloat16, seed=22))
    g = torch.Generator().manual_seed(23)
    q, nk, nv = (torch.zeros(2, h, tokens, 64, dtype=torch.bfloat16, device=DEV) for h in (4, 2, 2))
    parents = torch.tensor([_tree(random.Random(z), tokens) for z in range(2)], dtype=torch.int32, device=DEV)
    path = torch.tensor([[0, 2, 3, 6], [1, 2, 4, 7]], dtype=torch.int32, device=DEV)
    counts = torch.tensor([4, 2], dtype=torch.int32, device=DEV)

    def step(k, v, n):
        cache.append(nk, nv, k, v, table, n)
        out = cache.tree_attention(q, k, v, table, n, parents, max_length=320)
        return out, cache.keep_path(k, v, table, n, path, counts)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step(k.clone(), v.clone(), n)
    torch.cuda.current_stream().wait_stream(warm)
    ek, ev, en = k.clone(), v.clone(), n.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, after = step(k, v, n)
    for _ in range(4):
        for t in (q, nk, nv):
            t.copy_(torch.randn(t.shape, generator=g).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        want, en2 = step(ek, ev, en)
        assert torch.equal(out, want) and torch.equal(after, en2)
        _equal(k, ek)
        n.copy_(after)
        en = en2


def test_two_streams_and_schemas():
    from aotriton_amd import cache
    k, v, table, n = (t.to(DEV) for t in _pool([2000, 30], 5, 2, 128, 64, torch.bfloat16, seed=24))
    q = torch.randn(2, 8, 5, 128, device=DEV).bfloat16()
    want = cache.tree_attention(q, k, v, table, n)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(cache.tree_attention(q, k, v, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)
    torch.library.opcheck(torch.ops.aotriton_amd.tree_attention, (q, k, v, table, n, None, 2000, 0, 0, 0.1),
                          test_utils=('test_schema', 'test_faketensor'))
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    for op, args in (('cache_append', (q[:, :2], q[:, :2], k, v, table, n, None)), ('cache_copy_pages', (k, v, one, one + 1)),
                     ('cache_keep_path', (k, v, table, n, torch.zeros(2, 1, dtype=torch.int32, device=DEV), n * 0))):
        torch.library.opcheck(getattr(torch.ops.aotriton_amd, op), args, test_utils=('test_schema', 'test_faketensor'))
    with pytest.raises(NotImplementedError, match='no gradient'):
        cache.tree_attention(q.requires_grad_(True), k, v, table, n)


def test_writes_are_seen_by_autograd():
    from aotriton_amd import cache
    k, v, table, n = (t.to(DEV) for t in _pool([20, 5], 4, 2, 64, 16, torch.float16, seed=82))
    new = torch.randn(2, 2, 4, 64, device=DEV).half()
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    uses = torch.ones(k.shape[0], dtype=torch.int32, device=DEV)
    calls = [(lambda: cache.append(new, new, k, v, table, n), (k, v)),
             (lambda: cache.copy_pages(k, v, ints(0), ints(1)), (k, v)),
             (lambda: cache.keep_path(k, v, table, n, ints(0, 1, 2, 3).view(2, 2), ints(1, 2)), (k, v)),
             (lambda: cache.fork(k, v, table, n, uses, ints(0), ints(1), ints(3)), (k, v, table, n, uses)),
             (lambda: cache.free(table, uses, ints(0), ints(0), ints(1)), (table, uses))]
    for call, written in calls:
        before = [t._version for t in written]
        call()
        assert [t._version for t in written] == [x + 1 for x in before]
    for quiet in (torch.no_grad, torch.inference_mode):
        with quiet():
            before = k._version
            calls[0][0]()
            assert k._version == before + 1
    with torch.inference_mode():
        mine = [t.clone() for t in (k, v)]
    cache.append(new, new, *mine, table, n)
    _equal(mine[0], k)
    # a backward that needs a cache as it was says so
    w = torch.ones_like(k, requires_grad=True)
    y = (w * k).sum()
    calls[0][0]()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()


@pytest.mark.parametrize('window', [0, 30])
def test_compiled_serving_step(window):
    from aotriton_amd import cache
    k, v, table, n = (t.to(DEV) for t in _pool([300, 45], 16, 2, 64, 16, torch.bfloat16, seed=83))
    g = torch.Generator().manual_seed(84)
    q, nk, nv = (torch.randn(2, 8, h, 64, generator=g).bfloat16().to(DEV).transpose(1, 2) for h in (4, 2, 2))
    parents = torch.tensor([_tree(random.Random(z), 8) for z in range(2)], dtype=torch.int32, device=DEV)
    path = torch.tensor([[0, 2, 3, 6], [1, 2, 4, 7]], dtype=torch.int32, device=DEV)
    counts = torch.tensor([4, 2], dtype=torch.int32, device=DEV)

    def step(k, v, n):
        cache.append(nk, nv, k, v, table, n)
        out, lse = cache.tree_attention(q, k, v, table, n, parents, max_length=320, window=window, sinks=2 if window else 0, return_lse=True)
        return out.transpose(1, 2).reshape(2, 8, 256), lse, cache.keep_path(k, v, table, n, path, counts)
    torch._dynamo.reset()
    compiled = torch.compile(step, backend='aot_eager', fullgraph=True)
    ek, ev, en, cn = k.clone(), v.clone(), n, n
    for _ in range(2):
        *want, en = step(ek, ev, en)
        *got, cn = compiled(k, v, cn)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(cn, en)
        _equal(k, ek)
        _equal(v, ev)
