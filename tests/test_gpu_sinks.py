"""Attention with a sliding window and sinks, forward and backward, against the 64-bit oracle: windows and sinks around the tiles' edges,
more queries than keys and the other way round, packed sequences, head dims that are rounded up, strides, streams, graphs.  The bounds
are those of tests/_longctx.py."""
import math

import pytest
import torch

from _longctx import assert_within, grad_bounds, lse_bound, out_bound, score_error
from oracle import longctx

pytestmark = pytest.mark.gpu

DEV = 'cuda'

CASES = [
    # B, Hq, Hk, Sq, Sk, D, window, sinks, dtype
    (1, 1, 1, 1, 1, 64, 1, 0, torch.bfloat16),
    (1, 2, 1, 1, 300, 128, 17, 3, torch.float16),                 # a single query
    (2, 4, 2, 331, 331, 64, 100, 4, torch.float16),
    (1, 4, 4, 700, 700, 128, 64, 1, torch.bfloat16),
    (1, 8, 2, 513, 513, 128, 1, 1, torch.bfloat16),               # itself and the first key
    (1, 2, 2, 600, 600, 128, 200, 64, torch.float16),             # sinks that end with a tile
    (1, 2, 2, 600, 600, 128, 130, 65, torch.bfloat16),
    (1, 2, 1, 900, 900, 64, 33, 300, torch.bfloat16),             # sinks over several tiles, most of them outside the window
    (1, 2, 2, 400, 400, 64, 1000, 4, torch.float16),              # a window that reaches past the start
    (1, 2, 2, 300, 300, 128, 40, 1024, torch.bfloat16),           # sinks beyond the keys
    (1, 3, 3, 257, 257, 128, 50, 0, torch.bfloat16),              # no sinks
    (1, 4, 1, 100, 1200, 128, 256, 8, torch.float16),             # a chunk behind earlier keys
    (2, 2, 2, 65, 640, 64, 31, 40, torch.bfloat16),
    (1, 2, 2, 300, 170, 64, 60, 5, torch.float16),                # queries before the first key
    (1, 2, 2, 40, 3, 128, 2, 1, torch.bfloat16),
    (1, 4, 2, 330, 330, 72, 90, 4, torch.bfloat16),               # head dims rounded up
    (1, 4, 2, 330, 330, 96, 90, 4, torch.float16),
    (1, 2, 1, 200, 200, 104, 48, 7, torch.bfloat16),
    (1, 2, 2, 200, 200, 40, 48, 7, torch.float16),
    (1, 16, 1, 150, 150, 64, 20, 2, torch.bfloat16),              # one key head
]


def _inputs(B, Hq, Hk, Sq, Sk, D, dtype, seed=0, Dv=None, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: (torch.randn(*s, generator=g) * scale).to(dtype).to(DEV)
    Dv = D if Dv is None else Dv
    # (batch, tokens, heads, head dim) storage
    return (rn(B, Sq, Hq, D).transpose(1, 2), rn(B, Sk, Hk, D).transpose(1, 2), rn(B, Sk, Hk, Dv).transpose(1, 2),
            rn(B, Sq, Hq, Dv).transpose(1, 2))


def _check(q, k, v, do, window, sinks, scale, out, lse, grads, what='', device='cpu'):
    """one sequence, (heads, rows, head dim)"""
    dt = q.dtype
    q, k, v, do = (t.detach().to(device) for t in (q, k, v, do))
    seen = longctx.sink_mask(q.shape[1], k.shape[1], window, sinks, device=device)
    want, want_lse, p = longctx.attention(q, k, v, seen, scale)
    size = torch.matmul(p, v.double().abs().repeat_interleave(q.shape[0] // k.shape[0], 0))
    e = score_error(q, k, scale)
    values = v.double().abs().sum(1, keepdim=True).repeat_interleave(q.shape[0] // k.shape[0], 0)
    assert_within(what + 'out', out, want, out_bound(dt, want, size, values, e))
    if lse is not None:
        assert_within(what + 'lse', lse, want_lse, lse_bound(torch.where(want_lse.isinf(), 0.0, want_lse), e))
    if grads is None:
        return
    wants = longctx.attention_grads(q, k, v, do, seen, scale)
    bounds = grad_bounds(dt, q, k, v, do, seen, scale, want, size, p)
    u, tiny = bounds[3:]
    for name, got, w, b in zip(('dq', 'dk', 'dv'), grads, wants, bounds):
        assert_within(what + name, got, w, b + u * w.abs() + tiny)


def _step(q, k, v, do, window, sinks, scale=None, **packed):
    from aotriton_amd import torch_ops
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = torch_ops.sink_attention(q, k, v, window, sinks, scale=scale, **packed)
    return out.detach(), torch.autograd.grad(out, (q, k, v), do)


def _raw(q, k, v, window, sinks, scale):
    return torch.ops.aotriton_amd.sink_attention_forward(q, k, v, None, None, 0, 0, window, sinks, scale)


@pytest.mark.parametrize('B,Hq,Hk,Sq,Sk,D,window,sinks,dtype', CASES)
def test_against_the_oracle(B, Hq, Hk, Sq, Sk, D, window, sinks, dtype):
    q, k, v, do = _inputs(B, Hq, Hk, Sq, Sk, D, dtype, seed=Sq + D)
    scale = 1 / math.sqrt(D)
    out, grads = _step(q, k, v, do, window, sinks)
    _, lse = _raw(q, k, v, window, sinks, scale)
    for b in range(B):
        _check(q[b], k[b], v[b], do[b], window, sinks, scale, out[b], lse.view(B, Hq, Sq)[b], [g[b] for g in grads], f'sequence {b} ')


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('D', [64, 128])
def test_packed_sequences(D, dtype):
    lens_q, lens_k = [1, 300, 0, 77, 513, 5], [1, 300, 7, 200, 513, 2]
    Hq, Hk, window, sinks = 4, 2, 70, 5
    tq, tk, pad = sum(lens_q), sum(lens_k), 3            # rows behind the last sequence
    q, _, _, do = _inputs(1, Hq, Hk, tq + pad, 1, D, dtype, seed=1)
    _, k, v, _ = _inputs(1, Hq, Hk, 1, tk + pad, D, dtype, seed=2)
    offs = lambda lens: [sum(lens[:i]) for i in range(len(lens) + 1)]
    cq, ck = offs(lens_q), offs(lens_k)
    cu = lambda o: torch.tensor(o, dtype=torch.int32, device=DEV)
    out, grads = _step(q, k, v, do, window, sinks, cu_seqlens_q=cu(cq), cu_seqlens_k=cu(ck), max_seqlen_q=max(lens_q), max_seqlen_k=max(lens_k))
    for i in range(len(lens_q)):
        sq, sk = slice(cq[i], cq[i + 1]), slice(ck[i], ck[i + 1])
        _check(q[0][:, sq], k[0][:, sk], v[0][:, sk], do[0][:, sq], window, sinks, 1 / math.sqrt(D), out[0][:, sq], None,
               [grads[0][0][:, sq], grads[1][0][:, sk], grads[2][0][:, sk]], f'sequence {i} ')


def test_rows_behind_the_last_sequence_stay():
    import ctypes
    from aotriton_amd._lib import fa_fwd_params, lib
    q, k, v, _ = _inputs(1, 2, 2, 200, 200, 64, torch.bfloat16)
    out = torch.full_like(q, 7.0)
    lse = torch.full((2, 200), 7.0, device=DEV)
    cu = torch.tensor([0, 90, 150], dtype=torch.int32, device=DEV)
    c = fa_fwd_params()
    for view, t in ((c.Q, q), (c.K, k), (c.V, v), (c.Out, out), (c.L, lse), (c.cu_seqlens_q, cu), (c.cu_seqlens_k, cu)):
        _view(view, t)
    c.Max_seqlen_q = c.Max_seqlen_k = 90
    c.varlen_type = 1
    c.Sm_scale = 0.125
    assert lib.fa_attn_fwd_sinks(ctypes.byref(c), 3, 30, 4, torch.cuda.current_stream().cuda_stream, None, None) == 0
    torch.cuda.synchronize()
    # (the logsumexp of packed sequences is (heads, tokens up to the last offset))
    flat = lse.flatten()
    assert (out[:, :, 150:] == 7).all() and (flat[2 * 150:] == 7).all()
    _check(q[0][:, :90], k[0][:, :90], v[0][:, :90], q[0][:, :90], 30, 4, 0.125, out[0][:, :90], flat[:2 * 150].view(2, 150)[:, :90], None)


def _view(view, t):
    view.ptr = t.data_ptr()
    for i in range(t.dim()):
        view.sizes[i] = t.shape[i]
        view.strides[i] = t.stride(i)
    from aotriton_amd.flash import cast_dtype
    view.dtype = int(cast_dtype(t.dtype))


def test_different_value_head_dim_and_strides():
    q, k, v, do = _inputs(2, 4, 2, 210, 260, 64, torch.float16, seed=5, Dv=96)
    k = torch.empty(2, 2, 520, 64, dtype=k.dtype, device=DEV)[:, :, ::2].copy_(k)      # every other row
    out, grads = _step(q, k, v, do, 77, 6)
    for b in range(2):
        _check(q[b], k[b], v[b], do[b], 77, 6, 0.125, out[b], None, [g[b] for g in grads])


def test_unaligned_and_shared_inputs():
    """rows that are no 16-byte pieces are copied; a key head that is expanded gets the sum of its gradients"""
    q, k, v, do = _inputs(1, 2, 2, 130, 130, 64, torch.bfloat16, seed=6)
    odd = torch.empty(1, 2, 130, 67, dtype=q.dtype, device=DEV)[..., 1:65].copy_(q)
    out, grads = _step(odd, k, v, do, 33, 4)
    _check(q[0], k[0], v[0], do[0], 33, 4, 0.125, out[0], None, [g[0] for g in grads])
    from aotriton_amd import torch_ops
    one = k[:, :1].detach().clone().requires_grad_(True)
    out = torch_ops.sink_attention(q, one.expand(1, 2, 130, 64), v, 33, 4)
    (got,) = torch.autograd.grad(out, one, do)
    two, grads = _step(q, k[:, :1].expand(1, 2, 130, 64), v, do, 33, 4)
    assert torch.equal(out, two)
    assert torch.equal(got, grads[1].sum(1, keepdim=True))


@pytest.mark.parametrize('D', [64, 128])
def test_the_lowest_and_the_largest_scores(D):
    """scores beyond exp's range both ways, rows whose sinks are all that counts or do not count at all"""
    q, k, v, do = _inputs(1, 2, 2, 300, 300, D, torch.bfloat16, seed=7, scale=1.0)
    k[:, :, :4] *= 60
    scale = 0.5
    out, grads = _step(q, k, v, do, 40, 4, scale=scale)
    _check(q[0], k[0], v[0], do[0], 40, 4, scale, out[0], None, [g[0] for g in grads])


def test_hidden_keys_may_be_anything():
    """keys that no query sees: between the sinks and a chunk's window"""
    q, k, v, do = _inputs(1, 2, 2, 64, 1024, 128, torch.float16, seed=8)
    want, grads = _step(q, k, v, do, 64, 4)
    k[:, :, 256:640] = float('nan')
    v[:, :, 256:640] = float('inf')
    out, grads2 = _step(q, k, v, do, 64, 4)
    assert torch.equal(out, want)
    for a, b in zip(grads, grads2):
        assert torch.equal(a, b)


def test_a_wide_window_is_causal_attention():
    from aotriton_amd import torch_ops
    q, k, v, _ = _inputs(2, 4, 2, 500, 500, 128, torch.bfloat16, seed=9)
    out = torch_ops.sink_attention(q, k, v, 2 ** 31 - 1, 0)
    ref = torch_ops.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)
    for b in range(2):
        _check(q[b], k[b], v[b], q[b], 500, 0, 1 / math.sqrt(128), out[b], None, None)
        _check(q[b], k[b], v[b], q[b], 500, 0, 1 / math.sqrt(128), ref[b], None, None)


@pytest.mark.parametrize('Sq,Sk', [(0, 0), (0, 5), (5, 0)])
def test_nothing_to_do(Sq, Sk):
    q, k, v, do = _inputs(1, 2, 2, Sq, Sk, 64, torch.bfloat16)
    out, grads = _step(q, k, v, do, 3, 1)
    assert out.shape == q.shape and (out == 0).all()
    for g, t in zip(grads, (q, k, v)):
        assert g.shape == t.shape and (g == 0).all()


def test_no_sequence_and_no_token():
    q, k, v, do = _inputs(0, 4, 2, 30, 40, 64, torch.bfloat16)
    out, grads = _step(q, k, v, do, 3, 1)
    assert out.shape == q.shape and [g.shape for g in grads] == [t.shape for t in (q, k, v)]
    q, k, v, do = _inputs(1, 4, 2, 5, 7, 64, torch.bfloat16)      # tokens that belong to no sequence
    cu = torch.zeros(3, dtype=torch.int32, device=DEV)
    out, grads = _step(q, k, v, do, 3, 1, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=1, max_seqlen_k=1)
    assert all((t == 0).all() for t in (out, *grads))


def test_results_do_not_change_and_other_streams():
    q, k, v, do = _inputs(2, 8, 2, 777, 777, 128, torch.bfloat16, seed=10)
    want = _step(q, k, v, do, 100, 4)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            got.append(_step(q, k, v, do, 100, 4))
    torch.cuda.synchronize()
    for out, grads in got:
        assert torch.equal(out, want[0])
        assert all(torch.equal(a, b) for a, b in zip(grads, want[1]))


def test_captured_step():
    """forward and backward in a graph, replayed on new values with eager work between the replays"""
    sets = [_inputs(1, 4, 2, 400, 400, 64, torch.float16, seed=20 + i) for i in range(3)]
    static = [t.clone() for t in sets[0]]
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        _step(*static, 90, 4)
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = _step(*static, 90, 4)
    for values in sets + sets[:1]:
        for s, x in zip(static, values):
            s.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = _step(*values, 90, 4)
        assert torch.equal(out, want[0])
        assert all(torch.equal(a, b) for a, b in zip(grads, want[1]))


def test_compiled_and_traced():
    from aotriton_amd import torch_ops
    q, k, v, do = _inputs(1, 2, 2, 100, 100, 64, torch.bfloat16, seed=11)
    torch.library.opcheck(torch.ops.aotriton_amd.sink_attention_forward, (q, k, v, None, None, 0, 0, 30, 4, 0.125),
                          test_utils=('test_schema', 'test_faketensor'))
    out, lse = _raw(q, k, v, 30, 4, 0.125)
    torch.library.opcheck(torch.ops.aotriton_amd.sink_attention_backward, (do, q, k, v, out, lse, None, None, 0, 0, 30, 4, 0.125),
                          test_utils=('test_schema', 'test_faketensor'))
    assert torch.equal(torch_ops.sink_attention(q, k, v, 30, 4), out)


def test_second_derivatives_are_refused():
    from aotriton_amd import torch_ops
    q, k, v, do = _inputs(1, 1, 1, 20, 20, 64, torch.bfloat16)
    q = q.detach().requires_grad_(True)
    out = torch_ops.sink_attention(q, k, v, 5, 1)
    (dq,) = torch.autograd.grad(out, q, do, create_graph=True)
    with pytest.raises(RuntimeError, match='second derivatives'):
        dq.sum().backward()


def test_the_library_takes_its_workspace_without_an_allocator():
    import ctypes
    from aotriton_amd._lib import fa_bwd_params, lib
    q, k, v, do = _inputs(1, 4, 2, 300, 300, 64, torch.bfloat16, seed=12)
    out, lse = _raw(q, k, v, 50, 4, 0.125)
    want = _step(q, k, v, do, 50, 4)[1]
    got = [torch.empty_like(t) for t in (q, k, v)]
    delta = torch.empty_like(lse)
    c = fa_bwd_params()
    for view, t in ((c.Q, q), (c.K, k), (c.V, v), (c.Out, out), (c.DO, do), (c.DQ, got[0]), (c.DK, got[1]), (c.DV, got[2]), (c.L, lse),
                    (c.D.eager, delta)):
        _view(view, t)
    c.Sm_scale = 0.125
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.fa_attn_bwd_sinks(ctypes.byref(c), 6, 50, 4, stream, None, None) == 0
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    lib.fa_set_bwd_workspace_limit(0)
    try:
        assert lib.fa_attn_bwd_sinks(ctypes.byref(c), 6, 50, 4, stream, None, None) == 2      # no memory, nothing launched
    finally:
        lib.fa_set_bwd_workspace_limit(-1)


@pytest.mark.parametrize('Hq,Hk,S,D,dtype', [
    (4, 1, 417, 128, torch.bfloat16), (8, 1, 290, 64, torch.float16), (6, 2, 333, 128, torch.float16), (12, 2, 200, 64, torch.bfloat16),
    (16, 2, 97, 128, torch.bfloat16), (7, 1, 130, 96, torch.float16), (8, 2, 33, 80, torch.bfloat16), (2, 1, 1000, 128, torch.bfloat16)])
def test_heads_of_a_group(Hq, Hk, S, D, dtype):
    """groups that take a workgroup's waves whole, in part, and not at all"""
    q, k, v, do = _inputs(2, Hq, Hk, S, S + 40, D, dtype, seed=S)
    out, grads = _step(q, k, v, do, 90, 5)
    _, lse = _raw(q, k, v, 90, 5, 1 / math.sqrt(D))
    for b in range(2):
        _check(q[b], k[b], v[b], do[b], 90, 5, 1 / math.sqrt(D), out[b], lse.view(2, Hq, S)[b], [g[b] for g in grads], f'sequence {b} ')


@pytest.mark.parametrize('Hq,Hk,S,window,D,dtype', [
    (32, 8, 4099, 1100, 128, torch.bfloat16), (32, 8, 4099, 1100, 96, torch.float16), (32, 8, 4099, 1100, 104, torch.bfloat16),
    (16, 16, 4100, 1030, 128, torch.float16), (32, 8, 4099, 1100, 64, torch.bfloat16),
    (32, 8, 8190, 1030, 128, torch.bfloat16), (32, 8, 8190, 1030, 104, torch.float16), (32, 32, 6000, 2900, 96, torch.bfloat16),
    (16, 4, 8190, 4100, 128, torch.float16), (16, 2, 8190, 4100, 104, torch.bfloat16), (12, 4, 8190, 4100, 96, torch.bfloat16)])
def test_long_sequences(Hq, Hk, S, window, D, dtype):
    """the kernels of long sequences (64 rows per wave above 64 columns); the oracle takes the first and the last group"""
    q, k, v, do = _inputs(1, Hq, Hk, S, S, D, dtype, seed=D)
    out, grads = _step(q, k, v, do, window, 40)
    _, lse = _raw(q, k, v, window, 40, 1 / math.sqrt(D))
    g = Hq // Hk
    for hk in (0, Hk - 1):
        hq, kv = slice(hk * g, hk * g + g), slice(hk, hk + 1)
        _check(q[0, hq], k[0, kv], v[0, kv], do[0, hq], window, 40, 1 / math.sqrt(D), out[0, hq], lse.view(Hq, S)[hq],
               [grads[0][0, hq], grads[1][0, kv], grads[2][0, kv]], f'group {hk} ', device=DEV)


@pytest.mark.parametrize('lens,Hq,Hk,D,sinks', [
    ([3, 1, 1000, 2] * 7 + [2900] + [1] * 60, 4, 1, 128, 70),          # one long one among many, three blocks of sinks
    ([1 + i * i % 37 for i in range(1100)] + [700], 2, 1, 64, 3),      # more sequences than a table holds
    ([5 + i % 11 for i in range(1100)], 2, 2, 128, 4),
    ([2500, 0, 0, 0, 1, 0], 8, 2, 128, 33)])
def test_sequences_of_very_different_lengths(lens, Hq, Hk, D, sinks):
    window, n = 50, sum(lens)
    q, k, v, do = _inputs(1, Hq, Hk, n, n, D, torch.bfloat16, seed=len(lens))
    offs = [0]
    for x in lens:
        offs.append(offs[-1] + x)
    cu = torch.tensor(offs, dtype=torch.int32, device=DEV)
    out, grads = _step(q, k, v, do, window, sinks, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=max(lens), max_seqlen_k=max(lens))
    assert all(torch.isfinite(t).all() for t in (out, *grads))
    for i in sorted({*range(0, len(lens), max(1, len(lens) // 24)), lens.index(max(lens)), len(lens) - 1}):
        at = slice(offs[i], offs[i + 1])
        _check(q[0][:, at], k[0][:, at], v[0][:, at], do[0][:, at], window, sinks, 1 / math.sqrt(D), out[0][:, at], None,
               [t[0][:, at] for t in grads], f'sequence {i} ', device=DEV)


@pytest.mark.parametrize('tail_q,tail_k,Hq,Hk,D,layout', [(5, 0, 4, 2, 64, 'tokens first'), (0, 300, 2, 2, 128, 'heads first'), (700, 1, 8, 1, 96, 'tokens first'),
                                                        (0, 0, 2, 1, 64, 'heads first')])
def test_tokens_behind_the_last_sequence_get_zeros(tail_q, tail_k, Hq, Hk, D, layout):
    lens = [130, 1, 77]
    n = sum(lens)
    q, _, _, do = _inputs(1, Hq, Hk, n + tail_q, 1, D, torch.float16, seed=50)
    _, k, v, _ = _inputs(1, Hq, Hk, 1, n + tail_k, D, torch.float16, seed=51)
    if layout == 'heads first':
        q, k, v, do = (t.contiguous() for t in (q, k, v, do))
    for t, tail in ((q, tail_q), (do, tail_q), (k, tail_k), (v, tail_k)):
        t[:, :, t.shape[2] - tail:] = float('nan')
    rubbish = [torch.full((1, Hq, n + 700, 128), float('nan'), dtype=torch.float16, device=DEV) for _ in range(8)]
    del rubbish      # what new tensors are made of
    cu = torch.tensor([0, 130, 131, n], dtype=torch.int32, device=DEV)
    out, grads = _step(q, k, v, do, 40, 3, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=130, max_seqlen_k=130)
    for t in (out, *grads):
        assert torch.isfinite(t).all() and (t[:, :, n:] == 0).all()
    at = slice(0, 130)
    _check(q[0][:, at], k[0][:, at], v[0][:, at], do[0][:, at], 40, 3, 1 / math.sqrt(D), out[0][:, at], None, [t[0][:, at] for t in grads])


@pytest.mark.parametrize('Hq,Hk,S,D,window,sinks', [(4, 2, 700, 64, 16, 4), (2, 2, 700, 128, 20, 70), (4, 1, 500, 96, 8, 0), (2, 1, 400, 64, 2, 1)])
def test_short_windows_take_delta_from_the_tiles(Hq, Hk, S, D, window, sinks):
    """With delta from P and dP in fp32 what is left of dQ's error are two roundings to 16 bits, of dS and of dQ.  One is off by u / m of the value,
    m the mantissa, evenly between -1 and 1 of it: u / sqrt(3) sqrt(E[1 / m^2]) = 0.425 u in the mean square (m spread as 1 / m: 3 / (8 ln 2)), two
    0.600 u.  4 % more for what is drawn; from the rounded output it is 0.65 u at a window of 16, 0.72 at 2."""
    q, k, v, do = _inputs(1, Hq, Hk, S, S, D, torch.float16, seed=60)
    _, grads = _step(q, k, v, do, window, sinks)
    seen = longctx.sink_mask(S, S, window, sinks, device=DEV)
    want = longctx.attention_grads(q[0], k[0], v[0], do[0], seen, 1 / math.sqrt(D))[0]
    off = ((grads[0][0].double() - want).norm() / want.norm()).item()
    assert off < 1.04 * 0.600 * 2.0 ** -11, off * 2 ** 11


def _odd(t, n=67):
    """the same values in (batch, tokens, heads, n) storage: rows that are no 16-byte pieces"""
    x = t.transpose(1, 2)
    return torch.empty(*x.shape[:3], n, dtype=t.dtype, device=t.device)[..., 1:1 + t.shape[3]].copy_(x).transpose(1, 2)


@pytest.mark.parametrize('which', ['q', 'k', 'v', 'all', 'offset'])
def test_layouts_of_results(which):
    """what the traced call says of its results' storage is what they have"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from aotriton_amd import torch_ops  # noqa: F401  (the fakes)
    q, k, v, do = _inputs(2, 4, 2, 130, 130, 64, torch.bfloat16, seed=80)
    if which == 'offset':
        q, k, v = (torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.transpose(1, 2).shape).copy_(t.transpose(1, 2)).transpose(1, 2) for t in (q, k, v))
    else:
        q, k, v = (_odd(t) if which in (name, 'all') else t for name, t in (('q', q), ('k', k), ('v', v)))
    fwd, bwd = torch.ops.aotriton_amd.sink_attention_forward, torch.ops.aotriton_amd.sink_attention_backward
    out, lse = fwd(q, k, v, None, None, 0, 0, 33, 4, 0.125)
    grads = bwd(do, q, k, v, out, lse, None, None, 0, 0, 33, 4, 0.125)
    with FakeTensorMode() as mode:
        f = [mode.from_tensor(t) for t in (do, q, k, v, out, lse)]
        said = [*fwd(*f[1:4], None, None, 0, 0, 33, 4, 0.125), *bwd(*f, None, None, 0, 0, 33, 4, 0.125)]
    for got, want in zip((out, lse, *grads), said):
        assert got.shape == want.shape and got.stride() == want.stride()


@pytest.mark.parametrize('packed', [False, True])
def test_compiled_steps_on_any_storage(packed):
    from aotriton_amd import torch_ops
    B = 1 if packed else 2
    q, k, v, do = _inputs(B, 4, 2, 130, 130, 64, torch.bfloat16, seed=81)
    extra = {}
    if packed:
        cu = torch.tensor([0, 70, 71, 130], dtype=torch.int32, device=DEV)
        extra = dict(cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=70, max_seqlen_k=70)

    def step(q, k, v):
        out = torch_ops.sink_attention(q, k, v, 33, 4, **extra)
        return out.transpose(1, 2).reshape(B, 130, 256)      # (a view, if the result is stored as the query is)
    weight = do.transpose(1, 2).reshape(B, 130, 256)
    want = None
    for odd in (False, True):
        leaves = [(_odd(t) if odd else t).detach().requires_grad_(True) for t in (q, k, v)]
        torch._dynamo.reset()
        compiled = torch.compile(step, backend='aot_eager', fullgraph=True)
        for f in (step, compiled):
            out = f(*leaves)
            got = (out.detach(), *torch.autograd.grad(out, leaves, weight))
            want = got if want is None else want
            assert all(torch.equal(a, b) for a, b in zip(got, want))
