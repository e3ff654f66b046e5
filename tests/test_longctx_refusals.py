"""What attention with sinks and the cache of pages refuse, on the host and before any HIP call, and the oracle that their GPU tests
compare with: its gradients against differences, its masks against a count."""
import ctypes
import math

import pytest
import torch

from oracle import longctx

INVALID, NOT_SUPPORTED, NO_GPU, SYMBOL, BACKEND = 1, 801, 209, 13, 217


def _lib():
    from aotriton_amd import _lib
    return _lib


def _code(dtype):
    from aotriton_amd.flash import cast_dtype
    return int(cast_dtype(dtype))


def _fill(view, sizes, dtype=torch.bfloat16, ptr=4096, strides=None):
    if strides is None:
        strides = [math.prod(sizes[i + 1:]) for i in range(len(sizes))]
    view.ptr = ptr
    for i, (n, s) in enumerate(zip(sizes, strides)):
        view.sizes[i], view.strides[i] = n, s
    view.dtype = _code(dtype)
    return view


def _fwd(D=64, dtype=torch.bfloat16, Sq=100, Sk=100, **change):
    L = _lib()
    p = L.fa_fwd_params()
    _fill(p.Q, (2, 4, Sq, D), dtype)
    _fill(p.K, (2, 2, Sk, D), dtype)
    _fill(p.V, (2, 2, Sk, D), dtype)
    _fill(p.Out, (2, 4, Sq, D), dtype)
    _fill(p.L, (8, Sq), torch.float32)
    p.Sm_scale = 1.0
    for name, value in change.items():
        setattr(p, name, value)
    return p


def _run_fwd(p, window=10, sinks=4, version=3, options=None):
    return _lib().lib.fa_attn_fwd_sinks(ctypes.byref(p), version, window, sinks, None, options, None)


ACCEPTED = (0, NO_GPU)      # (the device is asked after the arguments: none here)


def test_sinks_refusals():
    if torch.cuda.is_available():
        pytest.skip('arguments stand for no memory')
    L = _lib()
    assert _run_fwd(_fwd()) in ACCEPTED
    assert _run_fwd(_fwd(D=128), sinks=0) in ACCEPTED
    assert _run_fwd(_fwd(D=72), window=2 ** 31 - 1, sinks=1024) in ACCEPTED
    for window, sinks in ((0, 4), (-1, 4), (10, -1), (-2 ** 31, 0)):
        assert _run_fwd(_fwd(), window, sinks) == INVALID
    assert _run_fwd(_fwd(), sinks=1025) == NOT_SUPPORTED
    assert _run_fwd(_fwd(), version=2) == SYMBOL
    assert _run_fwd(_fwd(causal_type=3)) == INVALID
    assert _run_fwd(_fwd(D=136)) == NOT_SUPPORTED
    assert _run_fwd(_fwd(D=60)) == NOT_SUPPORTED
    assert _run_fwd(_fwd(dtype=torch.float32)) == NOT_SUPPORTED
    p = _fwd(dropout_p=0.1)
    p.philox_seed_ptr.ptr = 4096
    assert _run_fwd(p) == NOT_SUPPORTED
    p = _fwd()
    _fill(p.B, (2, 4, 100, 100))
    assert _run_fwd(p) == NOT_SUPPORTED
    p = _fwd()
    _fill(p.encoded_softmax, (2, 4, 100, 100))
    assert _run_fwd(p) == NOT_SUPPORTED
    p = _fwd()
    p.Q.ptr = 4098
    assert _run_fwd(p) == NOT_SUPPORTED
    p = _fwd()
    p.K.strides[2] = 65
    assert _run_fwd(p) == NOT_SUPPORTED
    p = _fwd()
    p.Out.sizes[2] = 99
    assert _run_fwd(p) == INVALID
    opt = L.fa_options(1, 0)
    assert _run_fwd(_fwd(), options=ctypes.byref(opt)) == BACKEND


def test_sinks_backward_refusals():
    if torch.cuda.is_available():
        pytest.skip('arguments stand for no memory')
    L = _lib()

    def params():
        p = L.fa_bwd_params()
        for name in ('Q', 'Out', 'DO', 'DQ'):
            _fill(getattr(p, name), (2, 4, 100, 64))
        for name in ('K', 'V', 'DK', 'DV'):
            _fill(getattr(p, name), (2, 2, 100, 64))
        _fill(p.L, (8, 100), torch.float32)
        _fill(p.D.eager, (8, 100), torch.float32)
        return p

    def run(p, window=10, sinks=4, options=None):
        return L.lib.fa_attn_bwd_sinks(ctypes.byref(p), 6, window, sinks, None, options, None)
    assert run(params()) in ACCEPTED
    assert run(params(), window=0) == INVALID
    assert run(params(), sinks=2000) == NOT_SUPPORTED
    p = params()
    p.causal_type = 3
    assert run(p) == INVALID
    p = params()
    p.D.eager.ptr = 0
    assert run(p) == BACKEND                       # without delta only a single launch could run
    assert run(params(), options=ctypes.byref(L.fa_options(1, 0))) == BACKEND
    p = params()
    p.DK.strides[2] = 63
    assert run(p) == NOT_SUPPORTED


def _cache(pages=9, heads=2, slots=16, D=64, Dv=None, dtype=torch.float16, sequences=3, columns=5):
    c = _lib().fa_cache()
    _fill(c.K, (pages, heads, slots, D), dtype)
    _fill(c.V, (pages, heads, slots, D if Dv is None else Dv), dtype)
    _fill(c.table, (sequences, columns), torch.int32)
    _fill(c.lengths, (sequences,), torch.int32)
    return c


def _tree(tokens=5, hq=4, **cache):
    p = _lib().fa_tree_params()
    p.cache = _cache(**cache)
    D, Dv = p.cache.K.sizes[3], p.cache.V.sizes[3]
    n = p.cache.lengths.sizes[0]
    dtype = cache.get('dtype', torch.float16)
    _fill(p.Q, (n, hq, tokens, D), dtype)
    _fill(p.Out, (n, hq, tokens, Dv), dtype)
    _fill(p.L, (n * hq, tokens), torch.float32)
    _fill(p.parents, (n, tokens), torch.int32)
    p.Sm_scale, p.max_length = 1.0, 50
    return p


def test_tree_refusals():
    if torch.cuda.is_available():
        pytest.skip('arguments stand for no memory')
    lib = _lib().lib

    def run(p=None, **change):
        p = _tree() if p is None else p
        for name, value in change.items():
            setattr(p, name, value)
        return lib.fa_tree_attn(ctypes.byref(p), None, None)
    for p in (_tree(), _tree(tokens=64), _tree(tokens=1, D=256, Dv=40), _tree(slots=1 << 20), _tree(columns=0), _tree(sequences=0, tokens=0)):
        assert run(p) in ACCEPTED
    assert lib.fa_tree_attn(None, None, None) == INVALID
    assert run(_tree(tokens=65)) == NOT_SUPPORTED
    for slots in (8, 24, 48, 1 << 21):
        assert run(_tree(slots=slots)) == NOT_SUPPORTED
    for D in (0, 60, 264):
        assert run(_tree(D=D)) == NOT_SUPPORTED
    assert run(_tree(dtype=torch.float32)) == INVALID
    assert run(_tree(hq=3)) == INVALID
    assert run(_tree(pages=0)) == INVALID
    assert run(_tree(columns=1 << 28)) == NOT_SUPPORTED                  # slots past 31 bits
    for change in (dict(window=-1), dict(sinks=-1), dict(sinks=3), dict(max_length=-1)):
        assert run(**change) == INVALID
    assert run(window=2 ** 31 - 1, sinks=2 ** 31 - 1) in ACCEPTED
    for change in (lambda p: setattr(p.cache.K, 'ptr', 0), lambda p: setattr(p.cache.lengths, 'ptr', 0), lambda p: setattr(p.cache.table, 'ptr', 0),
                   lambda p: setattr(p.Q, 'ptr', 0), lambda p: p.Q.sizes.__setitem__(0, 2), lambda p: p.Out.sizes.__setitem__(3, 72),
                   lambda p: p.cache.V.sizes.__setitem__(0, 8), lambda p: p.cache.table.sizes.__setitem__(0, 2),
                   lambda p: p.parents.sizes.__setitem__(1, 4), lambda p: setattr(p.parents, 'dtype', 13), lambda p: p.L.sizes.__setitem__(0, 11),
                   lambda p: setattr(p.cache.table, 'dtype', 13), lambda p: setattr(p.Q, 'dtype', 3)):
        p = _tree()
        change(p)
        assert run(p) == INVALID
    for change in (lambda p: setattr(p.cache.K, 'ptr', 4104), lambda p: p.cache.K.strides.__setitem__(3, 2), lambda p: p.cache.V.strides.__setitem__(2, 60),
                   lambda p: p.cache.V.strides.__setitem__(0, 2 ** 64 - 64), lambda p: p.cache.K.strides.__setitem__(0, 2 ** 31), lambda p: p.cache.table.strides.__setitem__(1, 2),
                   lambda p: p.cache.lengths.strides.__setitem__(0, 2), lambda p: p.Q.strides.__setitem__(1, 100), lambda p: p.L.strides.__setitem__(0, 9)):
        p = _tree()
        change(p)
        assert run(p) == NOT_SUPPORTED
    p = _tree()
    p.parents.ptr = p.L.ptr = 0
    assert run(p) in ACCEPTED


def test_page_refusals():
    if torch.cuda.is_available():
        pytest.skip('arguments stand for no memory')
    L = _lib()
    lib, ref = L.lib, ctypes.byref
    t1 = lambda n, dtype=torch.int32, ptr=4096: _fill(L.fa_tensor1(), (n,), dtype, ptr)
    t4 = lambda *s, dtype=torch.float16: _fill(L.fa_tensor4(), s, dtype)
    c = _cache()
    k, v = t4(3, 2, 7, 64), t4(3, 2, 7, 64)
    assert lib.fa_cache_append(ref(k), ref(v), ref(c), None, None) in ACCEPTED
    assert lib.fa_cache_append(ref(k), ref(v), ref(c), ref(t1(3)), None) in ACCEPTED
    assert lib.fa_cache_append(ref(k), ref(v), ref(c), ref(t1(2)), None) == INVALID
    assert lib.fa_cache_append(ref(k), None, ref(c), None, None) == INVALID
    assert lib.fa_cache_append(ref(k), ref(v), None, None, None) == INVALID
    for other in (t4(2, 2, 7, 64), t4(3, 1, 7, 64), t4(3, 2, 6, 64), t4(3, 2, 7, 72), t4(3, 2, 7, 64, dtype=torch.bfloat16)):
        assert lib.fa_cache_append(ref(k), ref(other), ref(c), None, None) == INVALID
    assert lib.fa_cache_copy_pages(ref(c.K), ref(c.V), ref(t1(4)), ref(t1(4)), None) in ACCEPTED
    assert lib.fa_cache_copy_pages(ref(c.K), ref(c.V), ref(t1(0, ptr=0)), ref(t1(0, ptr=0)), None) in ACCEPTED
    assert lib.fa_cache_copy_pages(ref(c.K), ref(c.V), ref(t1(4)), ref(t1(5)), None) == INVALID
    assert lib.fa_cache_copy_pages(ref(c.K), ref(c.V), ref(t1(4, torch.int64)), ref(t1(4)), None) == INVALID
    assert lib.fa_cache_copy_pages(ref(c.K), ref(c.V), ref(t1(4, ptr=0)), ref(t1(4)), None) == INVALID
    fork = lambda uses=9, n=2, cache=c: lib.fa_cache_fork(ref(cache), ref(t1(uses)), ref(t1(2)), ref(t1(n)), ref(t1(2)), None)
    assert fork() in ACCEPTED
    assert fork(uses=8) == INVALID and fork(n=3) == INVALID
    over = _cache()
    over.table.strides[0] = 4                       # rows that overlap
    assert fork(cache=over) == NOT_SUPPORTED
    path = _fill(L.fa_tensor2(), (3, 4), torch.int32)
    new = t1(3, ptr=8192)
    assert lib.fa_cache_keep_path(ref(c), ref(path), ref(t1(3)), ref(new), None) in ACCEPTED
    assert lib.fa_cache_keep_path(ref(c), ref(path), ref(t1(3)), ref(t1(3)), None) == INVALID      # onto the lengths themselves
    assert lib.fa_cache_keep_path(ref(c), ref(path), ref(t1(4)), ref(new), None) == INVALID
    assert lib.fa_cache_keep_path(ref(c), ref(_fill(L.fa_tensor2(), (2, 4), torch.int32)), ref(t1(3)), ref(new), None) == INVALID
    for which, dim in (('K', 0), ('V', 1), ('K', 2)):      # a cache that is expanded is read, not written
        wide = _cache()
        getattr(wide, which).strides[dim] = 0
        assert lib.fa_cache_append(ref(k), ref(v), ref(wide), None, None) == NOT_SUPPORTED
        assert lib.fa_cache_copy_pages(ref(wide.K), ref(wide.V), ref(t1(4)), ref(t1(4)), None) == NOT_SUPPORTED
        assert lib.fa_cache_keep_path(ref(wide), ref(path), ref(t1(3)), ref(new), None) == NOT_SUPPORTED
        assert fork(cache=wide) == NOT_SUPPORTED
        tree = _tree()
        tree.cache = wide
        assert lib.fa_tree_attn(ref(tree), None, None) in ACCEPTED
    table = _fill(L.fa_tensor2(), (3, 5), torch.int32)
    assert lib.fa_cache_free(ref(table), ref(t1(9)), ref(t1(2)), ref(t1(2)), ref(t1(2)), None) in ACCEPTED
    assert lib.fa_cache_free(ref(table), ref(t1(9)), ref(t1(2)), ref(t1(1)), ref(t1(2)), None) == INVALID
    assert lib.fa_cache_free(ref(over.table), ref(t1(9)), ref(t1(2)), ref(t1(2)), ref(t1(2)), None) == NOT_SUPPORTED


def test_tail_refusals():
    if torch.cuda.is_available():
        pytest.skip('arguments stand for no memory')
    L = _lib()

    def run(count=2, sizes=(1, 4, 100, 64), dtype=torch.bfloat16, ptr=4096, strides=None, cu=torch.int32, cu_ptr=4096, n=3):
        t, c = (L.fa_tensor4 * 2)(), (L.fa_tensor1 * 2)()
        for i in range(2):
            _fill(t[i], sizes, dtype, ptr, strides)
            _fill(c[i], (n,), cu, cu_ptr)
        return L.lib.fa_zero_tails(t, c, count, None)
    assert run() in ACCEPTED and run(count=0) in ACCEPTED and run(sizes=(1, 4, 0, 64), ptr=0) in ACCEPTED
    for bad in (dict(count=5), dict(count=-1), dict(sizes=(2, 4, 100, 64)), dict(dtype=torch.float32), dict(ptr=0), dict(cu=torch.int64), dict(cu_ptr=0), dict(n=0)):
        assert run(**bad) == INVALID
    for bad in (dict(sizes=(1, 4, 100, 60)), dict(ptr=4104), dict(strides=(1, 6400, 0, 1)), dict(strides=(1, 6404, 64, 1)), dict(strides=(1, 6400, 64, 2))):
        assert run(**bad) == NOT_SUPPORTED
    assert L.lib.fa_zero_tails(None, None, 1, None) == INVALID


# ---- the oracle -----------------------------------------------------------------------------------------------------

def test_mask_of_window_and_sinks():
    for sq, sk, window, sinks in ((5, 5, 2, 1), (1, 7, 3, 2), (6, 2, 1, 4), (4, 9, 100, 0)):
        seen = longctx.sink_mask(sq, sk, window, sinks)
        for i in range(sq):
            p = i + sk - sq
            assert seen[i].tolist() == [c <= p and (c > p - window or c < sinks) for c in range(sk)]


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(h, n, 5, generator=g, dtype=torch.float64) for h, n in ((4, 7), (2, 9), (2, 9), (4, 7)))
    seen = longctx.sink_mask(7, 9, 3, 2)
    f = lambda *t: float((longctx.attention(*t, seen, 0.4)[0] * do).sum())
    grads = longctx.attention_grads(q, k, v, do, seen, 0.4)
    h = 1e-5                                        # central differences: off by h^2 f''' / 6 and 2^-53 f / h
    for i in range(3):
        for _ in range(20):
            step = torch.randn(*(q, k, v)[i].shape, generator=g, dtype=torch.float64)
            at = lambda s: [t + s * h * step if j == i else t for j, t in enumerate((q, k, v))]
            assert abs((f(*at(1)) - f(*at(-1))) / (2 * h) - float((grads[i] * step).sum())) < 1e-7


def test_rows_without_a_key():
    seen = longctx.sink_mask(4, 2, 2, 1)
    q, k = torch.ones(1, 4, 3), torch.ones(1, 2, 3)
    out, lse, _ = longctx.attention(q, k, k, seen, 1.0)
    assert (out[0, :2] == 0).all() and torch.isinf(lse[0, :2]).all() and torch.isfinite(lse[0, 2:]).all()
    dq, dk, dv = longctx.attention_grads(q, k, k, q, seen, 1.0)
    assert torch.isfinite(dk).all() and (dq[0, :2] == 0).all()


def test_tree_masks():
    parents = [-1, 0, 0, 1, -1, 9, 5, 2]
    seen = longctx.tree_mask(3, 8, parents, 0, 0)
    drafted = [[0], [0, 1], [0, 2], [0, 1, 3], [4], None, None, [0, 2, 7]]
    for t, kin in enumerate(drafted):
        assert [s for s in range(11) if seen[t, s]] == ([] if kin is None else [0, 1, 2] + [3 + j for j in kin])
    seen = longctx.tree_mask(3, 8, parents, 2, 1)
    assert [s for s in range(11) if seen[3, s]] == [0, 3 + 1, 3 + 3]      # position 5: 4 and 5, and the sink


def test_host_checks_of_the_ops():
    from aotriton_amd import cache, torch_ops
    meta = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device='meta')
    assert torch_ops.sink_attention(meta(2, 4, 9, 64), meta(2, 2, 11, 64), meta(2, 2, 11, 32), 5, 2).shape == (2, 4, 9, 32)
    with pytest.raises(ValueError, match='neither'):
        torch_ops.sink_attention(meta(1, 4, 9, 64), meta(1, 2, 9, 64), meta(1, 2, 9, 64), 5, 2, cu_seqlens_q=meta(2))
    with pytest.raises(ValueError, match='max_seqlen'):
        torch_ops.sink_attention(meta(1, 4, 9, 64), meta(1, 2, 9, 64), meta(1, 2, 9, 64), 5, 2, cu_seqlens_q=meta(2), cu_seqlens_k=meta(2))
    out, lse = cache.tree_attention(meta(3, 4, 5, 64), meta(9, 2, 16, 64), meta(9, 2, 16, 64), meta(3, 4, dtype=torch.int32),
                                    meta(3, dtype=torch.int32), return_lse=True)
    assert out.shape == (3, 4, 5, 64) and lse.shape == (3, 4, 5)


def test_writes_to_a_cache_have_no_gradient():
    """where autograd would record one they say so, before any kernel"""
    from aotriton_amd import cache
    x = lambda grad=False: torch.zeros(3, 2, 16, 64, requires_grad=grad)
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32)
    calls = [lambda *t: cache.append(*t, ints(3, 1), ints(3)), lambda k, v, *_: cache.copy_pages(k, v, ints(1), ints(1)),
             lambda k, v, *_: cache.keep_path(k, v, ints(3, 1), ints(3), ints(3, 1), ints(3)),
             lambda k, v, *_: cache.fork(k, v, ints(3, 1), ints(3), ints(3), ints(1), ints(1), ints(1))]
    for call in calls:
        for i in range(4 if call is calls[0] else 2):
            with pytest.raises(NotImplementedError, match='no gradient'):
                call(*(x(j == i) for j in range(4)))
            with torch.no_grad(), pytest.raises(NotImplementedError, match='CPU'):      # (there is no kernel for this device)
                call(*(x(j == i) for j in range(4)))
