"""What latent attention, its cache and a batch's bookkeeping refuse, on the host and before any HIP call, and the oracle that their GPU tests compare
with: its gradients against differences, its two forms against each other."""
import ctypes
import math

import pytest
import torch

from oracle import latent

INVALID, NOT_SUPPORTED, NO_GPU = 1, 801, 209
ACCEPTED = (0, NO_GPU)      # (the device is asked after the arguments: none here)


def _lib():
    from aotriton_amd import _lib
    return _lib


def _fill(view, sizes, dtype=torch.bfloat16, ptr=4096, strides=None):
    from aotriton_amd.flash import cast_dtype
    if strides is None:
        strides = [math.prod(sizes[i + 1:]) for i in range(len(sizes))]
    view.ptr = ptr
    for i, (n, s) in enumerate(zip(sizes, strides)):
        view.sizes[i], view.strides[i] = n, s
    view.dtype = int(cast_dtype(dtype))
    return view


@pytest.fixture(autouse=True)
def no_gpu():
    if torch.cuda.is_available():
        pytest.skip('arguments stand for no memory')


def _fwd(B=2, H=3, Sq=50, Sk=70, E=64, R=32, Ev=64, dtype=torch.bfloat16, packed=0, p=None):
    p = _lib().fa_latent_fwd_params() if p is None else p
    for name, sizes in (('Q', (B, H, Sq, E + R)), ('K', (B, H, Sk, E)), ('V', (B, H, Sk, Ev)), ('S', (B, 1, Sk, R)), ('Out', (B, H, Sq, Ev))):
        _fill(getattr(p, name), sizes, dtype)
    _fill(p.L, (B * H, Sq), torch.float32)
    if packed:
        _fill(p.cu_seqlens_q, (packed + 1,), torch.int32)
        _fill(p.cu_seqlens_k, (packed + 1,), torch.int32)
        p.max_seqlen_q = p.max_seqlen_k = 50
    p.Sm_scale, p.causal = 0.1, 1
    return p


def _bwd(**kw):
    p = _lib().fa_latent_bwd_params()
    _fwd(p=p.fwd, **kw)
    for name, like in (('DO', p.fwd.Out), ('DQ', p.fwd.Q), ('DK', p.fwd.K), ('DV', p.fwd.V), ('DS', p.fwd.S)):
        _fill(getattr(p, name), list(like.sizes), kw.get('dtype', torch.bfloat16))
    return p


def _set(path, i, value):
    def f(p):
        *head, last = path.split('.')
        for name in head:
            p = getattr(p, name)
        if i is None:
            setattr(p, last, value)
        else:
            getattr(p, last)[i] = value
    return f


def test_expanded_refusals():
    run = lambda p: _lib().lib.fa_latent_fwd(ctypes.byref(p), None, None)
    for p in (_fwd(), _fwd(E=128, R=64, Ev=128), _fwd(E=8, R=8, Ev=8), _fwd(B=1, packed=3), _fwd(B=0), _fwd(Sq=0), _fwd(Sk=0), _fwd(E=72, R=16, Ev=128)):
        assert run(p) in ACCEPTED
    assert _lib().lib.fa_latent_fwd(None, None, None) == INVALID
    for p in (_fwd(E=136), _fwd(R=72), _fwd(Ev=136), _fwd(E=60), _fwd(R=4), _fwd(Ev=0), _fwd(H=65537)):
        assert run(p) == NOT_SUPPORTED
    assert run(_fwd(dtype=torch.float32)) == INVALID
    for change in (_set('K.ptr', None, 0), _set('S.ptr', None, 0), _set('S.sizes', 1, 3), _set('S.sizes', 2, 71), _set('K.sizes', 1, 2), _set('V.sizes', 2, 60), _set('V.sizes', 0, 1),
                   _set('Q.sizes', 3, 88), _set('Out.sizes', 2, 49), _set('Out.sizes', 3, 56), _set('K.dtype', None, 2), _set('L.sizes', 0, 5), _set('L.dtype', None, 2)):
        p = _fwd()
        change(p)
        assert run(p) == INVALID
    for change in (_set('Q.ptr', None, 4104), _set('K.strides', 3, 2), _set('V.strides', 2, 60), _set('S.strides', 2, 2 ** 64 - 32), _set('Q.strides', 2, (1 << 21) + 8),
                   _set('Out.strides', 2, 32), _set('Out.strides', 1, 0), _set('L.strides', 0, 51)):
        p = _fwd()
        change(p)
        assert run(p) == NOT_SUPPORTED
    for change in (_set('Q.strides', 2, 0), _set('K.strides', 1, 0), _set('L.ptr', None, 0)):      # read only; not wanted
        p = _fwd()
        change(p)
        assert run(p) in ACCEPTED
    for change in (_set('cu_seqlens_k.ptr', None, 0), _set('cu_seqlens_k.sizes', 0, 3), _set('cu_seqlens_q.dtype', None, 13), _set('cu_seqlens_q.strides', 0, 2), _set('max_seqlen_q', None, -1)):
        p = _fwd(B=1, packed=3)
        change(p)
        assert run(p) == INVALID
    assert run(_fwd(B=2, packed=3)) == INVALID


def test_expanded_backward_refusals():
    run = lambda p: _lib().lib.fa_latent_bwd(ctypes.byref(p), None, None)
    assert run(_bwd()) in (2, NO_GPU)               # (without scratch memory, where there is a device)
    assert _lib().lib.fa_latent_bwd(None, None, None) == INVALID
    for change in (_set('fwd.L.ptr', None, 0), _set('DO.sizes', 2, 49), _set('DQ.sizes', 3, 88), _set('DS.sizes', 2, 71), _set('DK.ptr', None, 0), _set('DV.dtype', None, 2)):
        p = _bwd()
        change(p)
        assert run(p) == INVALID
    for change in (_set('DQ.strides', 2, 8), _set('DK.strides', 1, 0), _set('DS.strides', 2, 0), _set('DV.ptr', None, 4104), _set('DO.strides', 3, 2)):
        p = _bwd()
        change(p)
        assert run(p) == NOT_SUPPORTED
    p = _bwd()
    p.DO.strides[2] = 0                             # a gradient that is the same for all rows is read only
    assert run(p) in (2, NO_GPU)


def _cache(rows=9, hq=4, pages=7, slots=16, E=576, Ev=512, sequences=3, columns=5, dtype=torch.float16):
    p = _lib().fa_latent_cache_params()
    _fill(p.Q, (1, rows, hq, E), dtype)
    _fill(p.Out, (1, rows, hq, Ev), dtype)
    _fill(p.L, (rows, hq), torch.float32)
    _fill(p.latent, (pages, 1, slots, E), dtype)
    _fill(p.table, (sequences, columns), torch.int32)
    _fill(p.lengths, (sequences,), torch.int32)
    _fill(p.starts, (sequences + 1,), torch.int32)
    p.Sm_scale, p.max_length = 0.1, 60
    return p


def test_absorbed_refusals():
    run = lambda p: _lib().lib.fa_latent_cache_attn(ctypes.byref(p), None, None)
    for p in (_cache(), _cache(E=8, Ev=8), _cache(slots=1 << 20), _cache(columns=0), _cache(sequences=0), _cache(rows=0), _cache(hq=128, rows=4000), _cache(E=320, Ev=8)):
        assert run(p) in ACCEPTED
    assert _lib().lib.fa_latent_cache_attn(None, None, None) == INVALID
    for slots in (8, 24, 1 << 21):
        assert run(_cache(slots=slots)) == NOT_SUPPORTED
    for p in (_cache(E=584), _cache(E=60, Ev=56), _cache(Ev=520), _cache(Ev=20), _cache(columns=1 << 28), _cache(hq=65537, rows=1)):
        assert run(p) == NOT_SUPPORTED
    for p in (_cache(E=64, Ev=72), _cache(dtype=torch.float32), _cache(pages=0), _cache(hq=0)):
        assert run(p) == INVALID
    for change in (_set('latent.ptr', None, 0), _set('latent.sizes', 1, 2), _set('Q.sizes', 3, 568), _set('Q.sizes', 0, 2), _set('Out.sizes', 2, 3), _set('table.sizes', 0, 2), _set('starts.sizes', 0, 3),
                   _set('lengths.dtype', None, 13), _set('L.sizes', 1, 5), _set('max_length', None, -1), _set('starts.ptr', None, 0), _set('Q.dtype', None, 3)):
        p = _cache()
        change(p)
        assert run(p) == INVALID
    for change in (_set('latent.ptr', None, 4104), _set('latent.strides', 3, 2), _set('latent.strides', 2, 580), _set('Q.strides', 1, 2 ** 64 - 576), _set('Q.strides', 1, 1 << 26), _set('Out.strides', 1, 0),
                   _set('table.strides', 1, 2), _set('starts.strides', 0, 2), _set('L.strides', 0, 5)):
        p = _cache()
        change(p)
        assert run(p) == NOT_SUPPORTED


def test_reserve_and_append_refusals():
    L = _lib()
    lib, ref = L.lib, ctypes.byref

    def reserve(n=3, columns=4, pages=9, tokens=20, slots=16):
        p = L.fa_reserve_params()
        _fill(p.table, (n, columns), torch.int32)
        for name, size in (('uses', pages), ('lengths', n), ('counts', n), ('starts', n + 1), ('missing', 1)):
            _fill(getattr(p, name), (size,), torch.int32)
        _fill(p.slot_map, (tokens,), torch.int64)
        p.slots = slots
        return p
    keep = ctypes.CFUNCTYPE(ctypes.c_void_p, ctypes.c_void_p, ctypes.c_uint64)(lambda self, n: None)

    class Allocator(ctypes.Structure):
        _fields_ = [('cookie', ctypes.c_void_p), ('alloc', type(keep))]
    alloc = Allocator(None, keep)
    run = lambda p: lib.fa_cache_reserve(ref(p), None, ctypes.cast(ctypes.pointer(alloc), ctypes.c_void_p))
    for p in (reserve(), reserve(n=0), reserve(tokens=0), reserve(pages=0), reserve(columns=0)):
        assert run(p) in (2, NO_GPU)
    assert lib.fa_cache_reserve(None, None, None) == INVALID and lib.fa_cache_reserve(ref(reserve()), None, None) == INVALID
    for slots in (0, 8, 24, 1 << 21):
        assert run(reserve(slots=slots)) == NOT_SUPPORTED
    for change in (_set('table.sizes', 0, 2), _set('counts.sizes', 0, 2), _set('starts.sizes', 0, 3), _set('missing.sizes', 0, 2), _set('slot_map.dtype', None, 12), _set('uses.ptr', None, 0),
                   _set('slot_map.ptr', None, 0)):
        p = reserve()
        change(p)
        assert run(p) == INVALID
    for change in (_set('table.strides', 0, 3), _set('table.strides', 1, 2), _set('uses.strides', 0, 2), _set('slot_map.strides', 0, 2)):
        p = reserve()
        change(p)
        assert run(p) == NOT_SUPPORTED

    t4 = lambda *s, dtype=torch.float16: _fill(L.fa_tensor4(), s, dtype)
    m = lambda n, dtype=torch.int64: _fill(L.fa_tensor1(), (n,), dtype)
    append = lambda k, v, kc, vc, s: lib.fa_cache_append_packed(ref(k), v and ref(v), kc and ref(kc), vc and ref(vc), ref(s), None)
    k, v, kc, vc = t4(1, 9, 2, 64), t4(1, 9, 2, 32), t4(7, 2, 16, 64), t4(7, 2, 16, 32)
    assert append(k, v, kc, vc, m(9)) in ACCEPTED and append(k, None, kc, None, m(9)) in ACCEPTED
    assert append(t4(1, 9, 1, 576), None, t4(7, 1, 16, 576), None, m(9)) in ACCEPTED
    assert append(t4(1, 0, 1, 576), None, t4(7, 1, 16, 576), None, m(0)) in ACCEPTED
    for args in ((k, v, kc, None, m(9)), (k, None, kc, vc, m(9)), (k, v, vc, kc, m(9)), (k, v, kc, vc, m(8)), (k, v, kc, vc, m(9, torch.int32)), (t4(2, 9, 2, 64), v, kc, vc, m(9)),
                 (t4(1, 9, 3, 64), v, kc, vc, m(9)), (k, t4(1, 8, 2, 32), kc, vc, m(9)), (t4(1, 9, 2, 64, dtype=torch.bfloat16), v, kc, vc, m(9)), (k, v, kc, None, m(9))):
        assert append(*args) == INVALID
    wide, flat = t4(7, 2, 16, 64), t4(7, 2, 16, 64)
    flat.strides[1] = 0
    wide.strides[3] = 2
    for kk, c in ((t4(1, 9, 2, 584), t4(7, 2, 16, 584)), (k, wide), (k, flat), (k, t4(7, 2, 24, 64))):
        assert append(kk, None, c, None, m(9)) == NOT_SUPPORTED


def test_host_checks_of_the_ops():
    from aotriton_amd import cache, torch_ops
    meta = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device='meta')
    ints = lambda *s: meta(*s, dtype=torch.int32)
    args = meta(2, 4, 9, 96), meta(2, 4, 11, 64), meta(2, 4, 11, 40), meta(2, 11, 32)
    assert torch_ops.latent_attention(*args).shape == (2, 4, 9, 40)
    with pytest.raises(ValueError, match='neither'):
        torch_ops.latent_attention(*args, cu_seqlens_q=ints(2))
    with pytest.raises(ValueError, match='max_seqlen'):
        torch_ops.latent_attention(*args, cu_seqlens_q=ints(2), cu_seqlens_k=ints(2))
    out, lse = cache.latent_attention(meta(7, 4, 576), meta(9, 1, 16, 576), ints(3, 4), ints(3), ints(4), 512, 0.1, return_lse=True)
    assert out.shape == (7, 4, 512) and lse.shape == (7, 4)
    starts, slots, missing = cache.reserve(ints(3, 4), ints(9), ints(3), ints(3), 7, 16)
    assert starts.shape == (4,) and slots.shape == (7,) and slots.dtype == torch.int64 and missing.shape == (1,)
    cache.append_packed(meta(7, 1, 576), None, meta(9, 1, 16, 576), None, meta(7, dtype=torch.int64))


def test_gap_refusals():
    """what fa_zero_gaps takes: as fa_zero_tails, and a greatest length for every tensor"""
    L = _lib()

    def run(count=2, sizes=(1, 4, 100, 64), dtype=torch.bfloat16, ptr=4096, strides=None, n=4, cu=torch.int32, cu_ptr=4096, longest=(50, 0)):
        t, c = (L.fa_tensor4 * 2)(), (L.fa_tensor1 * 2)()
        for i in range(2):
            _fill(t[i], sizes, dtype, ptr, strides)
            _fill(c[i], (n,), cu, cu_ptr)
        return L.lib.fa_zero_gaps(t, c, longest and (ctypes.c_int32 * 2)(*longest), count, None)
    assert run() in ACCEPTED and run(count=0) in ACCEPTED and run(sizes=(1, 4, 0, 64), ptr=0) in ACCEPTED and run(n=1) in ACCEPTED and run(count=0, longest=None) in ACCEPTED
    for bad in (dict(count=5), dict(count=-1), dict(sizes=(2, 4, 100, 64)), dict(dtype=torch.float32), dict(ptr=0), dict(cu=torch.int64), dict(cu_ptr=0), dict(n=0), dict(n=2 ** 31),
                dict(longest=None), dict(longest=(5, -1))):
        assert run(**bad) == INVALID
    for bad in (dict(sizes=(1, 4, 100, 60)), dict(ptr=4104), dict(strides=(1, 6400, 0, 1)), dict(strides=(1, 6404, 64, 1)), dict(strides=(1, 6400, 64, 2))):
        assert run(**bad) == NOT_SUPPORTED
    assert L.lib.fa_zero_gaps(None, None, None, 1, None) == INVALID


def test_writes_to_a_cache_have_no_gradient():
    from aotriton_amd import cache
    x = lambda grad=False: torch.zeros(3, 2, 16, 64, requires_grad=grad)
    r = lambda grad=False: torch.zeros(5, 2, 64, requires_grad=grad)
    slots = torch.zeros(5, dtype=torch.int64)
    for i in range(4):
        made = [f(j == i) for j, f in enumerate((r, r, x, x))]
        with pytest.raises(NotImplementedError, match='no gradient'):
            cache.append_packed(*made, slots)
        with torch.no_grad(), pytest.raises(NotImplementedError, match='CPU'):
            cache.append_packed(*made, slots)
    q, c = torch.zeros(2, 4, 64, requires_grad=True), torch.zeros(3, 1, 16, 64)
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32)
    for a, b in ((q, c), (q.detach(), c.requires_grad_(True))):
        with pytest.raises(NotImplementedError, match='no gradient'):
            cache.latent_attention(a, b, ints(1, 1), ints(1), ints(2), 64, 1.0)


# ---- the oracle ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('sq,sk,causal', [(5, 5, True), (3, 7, True), (6, 4, True), (4, 5, False)])
def test_gradients_against_differences(sq, sk, causal):
    g = torch.Generator().manual_seed(sq)
    rn = lambda *s: torch.randn(*s, dtype=torch.float64, generator=g)
    x = [rn(2, sq, 7), rn(2, sk, 4), rn(2, sk, 3), rn(sk, 3)]
    do = rn(2, sq, 3)
    grads = latent.attention_grads(*x, do, causal, 0.7)
    f = lambda x: float((latent.attention(*x, causal, 0.7)[0] * do).sum())
    for i, t in enumerate(x):
        d = rn(*t.shape)
        at = lambda h: f([y + h * d if j == i else y for j, y in enumerate(x)])
        assert abs((at(1e-5) - at(-1e-5)) / 2e-5 - float((grads[i] * d).sum())) < 1e-7


def test_the_two_forms_are_one():
    g = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(*s, dtype=torch.float64, generator=g)
    n, H, L, R, E, Ev, slots = 11, 3, 8, 4, 5, 6, 4
    w_k, w_v, rows, q = rn(H, L, E), rn(H, L, Ev), rn(n, L + R), rn(n, H, E + R)
    k, v = torch.einsum('nl,hle->hne', rows[:, :L], w_k), torch.einsum('nl,hle->hne', rows[:, :L], w_v)
    want = latent.attention(q.transpose(0, 1), k, v, rows[:, L:], True, 0.3)[0].transpose(0, 1)
    table, uses, starts, slot_map, missing = latent.reserve([[-1] * 5], [1, 0, 1, 0, 0], [0], [n], n, slots)
    assert missing == 0 and table == [[1, 3, 4, -1, -1]] and slot_map == [4, 5, 6, 7, 12, 13, 14, 15, 16, 17, 18]
    cache = torch.full((5, 1, slots, L + R), math.nan, dtype=torch.float64)
    for s, r in zip(slot_map, rows):
        cache[s // slots, 0, s % slots] = r
    absorbed = torch.cat([torch.einsum('nhe,hle->nhl', q[..., :E], w_k), q[..., E:]], 2)
    out, _, _ = latent.cache_attention(absorbed, cache, torch.tensor(table), torch.tensor([0]), torch.tensor(starts), L, 0.3)
    assert torch.allclose(torch.einsum('nhl,hle->nhe', out, w_v), want, atol=1e-12)


def test_reserve_of_a_short_pool():
    table, uses, starts, slot_map, missing = latent.reserve([[2, -1], [-1, -1], [0, -1]], [1, 0, 1], [3, 0, 4], [2, 3, -1], 4, 4)
    assert table == [[2, 1], [-1, -1], [0, -1]] and uses == [1, 1, 1] and starts == [0, 2, 4, 4] and slot_map == [11, 4, -1, -1] and missing == 1
