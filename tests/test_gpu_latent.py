"""Attention over keys that are part per head, part shared by all heads, forward and backward, against the 64-bit oracle: lengths around the
tiles' edges, one row to many, queries without a key, keys cut into parts, packed sequences, columns that are rounded up, strides, streams,
graphs.  The bounds are those of tests/_longctx.py; the shared part's gradient has those of its heads together, and of their fp32 sum."""
import math

import pytest
import torch

from _longctx import assert_within, grad_bounds, lse_bound, out_bound, score_error
from oracle import latent

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF, HF = torch.bfloat16, torch.float16

CASES = [
    # B, H, Sq, Sk, E, R, Ev, causal, dtype
    (1, 1, 1, 1, 128, 64, 128, True, BF),
    (1, 2, 1, 65, 64, 32, 64, True, HF),
    (2, 3, 64, 64, 128, 64, 128, True, HF),
    (1, 2, 127, 127, 128, 64, 128, True, BF),
    (1, 2, 129, 129, 64, 64, 64, True, BF),
    (2, 4, 331, 331, 64, 32, 64, True, HF),
    (1, 3, 257, 257, 128, 64, 128, False, BF),
    (1, 2, 200, 333, 128, 64, 128, True, HF),       # a chunk behind earlier keys
    (1, 2, 33, 700, 64, 64, 64, False, BF),
    (1, 2, 300, 170, 128, 64, 128, True, BF),       # queries before the first key
    (1, 2, 200, 3, 64, 8, 64, True, HF),
    (1, 2, 150, 150, 40, 24, 56, True, BF),         # columns that are rounded up
    (1, 2, 150, 150, 8, 8, 8, True, HF),
    (1, 2, 150, 150, 96, 32, 96, True, HF),
    (1, 2, 140, 140, 72, 16, 128, True, BF),
    (1, 2, 140, 140, 128, 40, 32, True, BF),
    (1, 1, 700, 700, 128, 64, 128, True, HF),
    (3, 5, 100, 100, 64, 32, 128, True, BF),
]


def _inputs(B, H, Sq, Sk, E, R, Ev, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)
    kv = rn(B, Sk, H, E + Ev).transpose(1, 2)       # as a projection leaves them
    return rn(B, Sq, H, E + R).transpose(1, 2), kv[..., :E], kv[..., E:], rn(B, Sk, R), rn(B, Sq, H, Ev).transpose(1, 2)


def _check(q, k, v, c, do, causal, scale, out, lse, grads, what=''):
    """one sequence, (heads, rows, columns); the shared part (rows, R)"""
    q, k, v, c, do = (t.detach().cpu() for t in (q, k, v, c, do))
    seen = latent.mask(q.shape[1], k.shape[1], causal)
    kk = latent.keys(k, c)
    want, want_lse, p = latent.attention(q, k, v, c, causal, scale)
    size = torch.matmul(p, v.double().abs())
    e = score_error(q, kk, scale)
    assert_within(what + 'out', out, want, out_bound(q.dtype, want, size, v.double().abs().sum(1, keepdim=True), e))
    if lse is not None:
        assert_within(what + 'lse', lse, want_lse, lse_bound(torch.where(want_lse.isinf(), 0.0, want_lse), e))
    if grads is None:
        return
    dq, dk, dv, dc = latent.attention_grads(q, k, v, c, do, causal, scale)
    bq, bk, bv, u, tiny = grad_bounds(q.dtype, q, kk, v, do, seen, scale, want, size, p)
    E, H = k.shape[2], q.shape[0]
    # A probability below the smallest number is 0 to the hardware (tests/_longctx.py: smallest): dS = P (dP - delta) is then off by that number
    # times |dP - delta|, which is 20 to 40 here, and the bounds count it once (scale 3: dK 5.3e-37 for 4.4e-37 where dP - delta is 30).
    lost = tiny * abs(scale) * torch.where(seen, (torch.matmul(do.double(), v.double().transpose(1, 2)) - (do.double() * want).sum(-1, keepdim=True)).abs(), 0.0)
    bq = bq + torch.matmul(lost, kk.double().abs())
    bk = bk + torch.matmul(lost.transpose(1, 2), q.double().abs())
    for name, got, w, b in (('dq', grads[0], dq, bq), ('dk', grads[1], dk, bk[..., :E]), ('dv', grads[2], dv, bv),
                            ('dshared', grads[3], dc, (1 + H * 2.0 ** -23) * bk[..., E:].sum(0))):
        assert_within(what + name, got, w, b + u * w.abs() + tiny)


def _step(q, k, v, c, do, causal=True, scale=None, **packed):
    from aotriton_amd import torch_ops
    q, k, v, c = (t.detach().requires_grad_(True) for t in (q, k, v, c))
    out = torch_ops.latent_attention(q, k, v, c, is_causal=causal, scale=scale, **packed)
    return out.detach(), torch.autograd.grad(out, (q, k, v, c), do)


def _raw(q, k, v, c, causal, scale):
    return torch.ops.aotriton_amd.latent_attention_forward(q, k, v, c, None, None, 0, 0, causal, scale)


@pytest.mark.parametrize('B,H,Sq,Sk,E,R,Ev,causal,dtype', CASES)
def test_against_the_oracle(B, H, Sq, Sk, E, R, Ev, causal, dtype):
    q, k, v, c, do = _inputs(B, H, Sq, Sk, E, R, Ev, dtype, seed=Sq + E)
    out, grads = _step(q, k, v, c, do, causal)
    _, lse = _raw(q, k, v, c, causal, 1 / math.sqrt(E + R))
    for b in range(B):
        _check(q[b], k[b], v[b], c[b], do[b], causal, 1 / math.sqrt(E + R), out[b], lse.view(B, H, Sq)[b], [g[b] for g in grads], f'sequence {b} ')


@pytest.mark.parametrize('dtype', [HF, BF])
def test_gradients_of_a_single_key(dtype):
    """P is 1 and dS = P (dP - delta) nothing, whatever O's rounding: what is left is P's error.  The logarithm of the sum, below 8 here, is rounded
    three times on its way, 3 2^-24 8, and the exponential and the product add less than as much again: dS is under 2^-18 |dP|.  (Delta from O
    in 16 bits is off by up to 2^-12 of its terms, 2^-8 for bf16.)  Half the smallest number that the type holds comes on top."""
    B, H, E, R, Ev = 3, 4, 128, 64, 128
    q, k, v, c, do = _inputs(B, H, 1, 1, E, R, Ev, dtype, seed=8)
    out, (dq, dk, _, dc) = _step(q, k, v, c, do, scale=0.05)
    assert torch.equal(out, v)
    assert (torch.matmul(q.float(), torch.cat([k, c[:, None].expand(-1, H, -1, -1)], -1).float().transpose(2, 3)) * 0.05 * 1.5).abs().max() < 8
    dp = (do.double() * v.double()).abs().sum(-1, keepdim=True)
    least = 2.0 ** -25 if dtype == HF else 0.0
    bound = 2.0 ** -18 * 0.05 * dp
    assert (dq[..., :E].double().abs() <= bound * k.double().abs() + least).all()
    assert (dq[..., E:].double().abs() <= bound * c[:, None].double().abs() + least).all()
    assert (dk.double().abs() <= bound * q[..., :E].double().abs() + least).all()
    assert (dc.double().abs() <= (bound * q[..., E:].double().abs()).sum(1) + least).all()


@pytest.mark.parametrize('dtype', [HF, BF])
@pytest.mark.parametrize('n', [2, 4, 21, 64])
def test_gradients_of_one_tile(n, dtype):
    """P and dS go through the products as two numbers of 16 bits each, off by u^2, and delta is the sum of P dP: what the gradients are off by is their
    own rounding, u, and what fp32 sums (fdot) and scores (e) leave."""
    B, H, E, R, Ev, scale = 2, 3, 128, 64, 128, 0.02
    q, k, v, c, do = _inputs(B, H, n, n, E, R, Ev, dtype, seed=n)
    _, grads = _step(q, k, v, c, do, scale=scale)
    for b in range(B):
        Q, K, V, C, DO = (t[b].cpu() for t in (q, k, v, c, do))
        kk = latent.keys(K, C)
        _, _, p = latent.attention(Q, K, V, C, True, scale)
        want = latent.attention_grads(Q, K, V, C, DO, True, scale)
        e, u, fdot = score_error(Q, kk, scale), torch.finfo(dtype).eps / 2, (E + R + 8) * 2.0 ** -24
        dp, dp_off = torch.matmul(DO.double(), V.double().transpose(1, 2)), fdot * torch.matmul(DO.double().abs(), V.double().abs().transpose(1, 2))
        share = 1.1 * u * u + 2 * e + (2 * n + 8) * 2.0 ** -24
        delta = (p * dp).sum(-1, keepdim=True)
        delta_off = (p * (share * dp.abs() + dp_off)).sum(-1, keepdim=True)
        off = share * (p * (dp - delta)).abs() + 1.01 * p * (dp_off + delta_off)
        least = 2.0 ** -24 if dtype == HF else 0.0      # (fp16's least number, for what is left of dS and P, and for the results)
        off, p_off = off + least, share * p + least
        bk = scale * torch.matmul(off.transpose(1, 2), Q.double().abs())
        for name, got, w, bound in (('dq', grads[0][b], want[0], scale * torch.matmul(off, kk.double().abs())), ('dk', grads[1][b], want[1], bk[..., :E]),
                                    ('dv', grads[2][b], want[2], torch.matmul(p_off.transpose(1, 2), DO.double().abs())), ('dshared', grads[3][b], want[3], bk[..., E:].sum(0))):
            assert_within(name, got, w, bound + u * w.abs() + least)


@pytest.mark.parametrize('B,H,Sq,Sk,E,R,Ev,causal,dtype', [
    (1, 1, 1, 4000, 128, 64, 128, True, BF), (1, 2, 130, 3000, 128, 64, 128, True, HF), (2, 1, 5, 2049, 64, 32, 64, False, HF),
    (1, 3, 17, 1100, 40, 8, 24, True, BF), (1, 1, 2000, 1900, 64, 64, 64, True, BF)])
def test_keys_cut_into_parts(B, H, Sq, Sk, E, R, Ev, causal, dtype):
    q, k, v, c, do = _inputs(B, H, Sq, Sk, E, R, Ev, dtype, seed=3)
    scale = 0.1
    out, lse = _raw(q, k, v, c, causal, scale)
    for b in range(B):
        _check(q[b], k[b], v[b], c[b], do[b], causal, scale, out[b], lse.view(B, H, Sq)[b], None)


@pytest.mark.parametrize('dtype', [HF, BF])
@pytest.mark.parametrize('E,R,Ev', [(64, 32, 64), (128, 64, 128), (72, 64, 40)])
@pytest.mark.parametrize('causal', [True, False])
def test_packed_sequences(E, R, Ev, causal, dtype):
    lens_q, lens_k = [1, 300, 0, 77, 513, 5, 40], [1, 300, 7, 200, 513, 2, 0]
    H, tq, tk, pad = 3, sum(lens_q), sum(lens_k), 3
    q, _, _, _, do = _inputs(1, H, tq + pad, 1, E, R, Ev, dtype, seed=1)
    _, k, v, c, _ = _inputs(1, H, 1, tk + pad, E, R, Ev, dtype, seed=2)
    for t in (q, do):
        t[:, :, tq:] = float('nan')                  # rows of no sequence may hold anything
    for t in (k, v):
        t[:, :, tk:] = float('inf')
    c[:, tk:] = float('nan')
    offs = lambda lens: [sum(lens[:i]) for i in range(len(lens) + 1)]
    cq, ck = offs(lens_q), offs(lens_k)
    cu = lambda o: torch.tensor(o, dtype=torch.int32, device=DEV)
    out, grads = _step(q, k, v, c, do, causal, cu_seqlens_q=cu(cq), cu_seqlens_k=cu(ck), max_seqlen_q=max(lens_q), max_seqlen_k=max(lens_k))
    for i in range(len(lens_q)):
        sq, sk = slice(cq[i], cq[i + 1]), slice(ck[i], ck[i + 1])
        _check(q[0][:, sq], k[0][:, sk], v[0][:, sk], c[0][sk], do[0][:, sq], causal, 1 / math.sqrt(E + R), out[0][:, sq], None,
               [grads[0][0][:, sq], grads[1][0][:, sk], grads[2][0][:, sk], grads[3][0][sk]], f'sequence {i} ')
    assert (out[:, :, tq:] == 0).all() and (grads[0][:, :, tq:] == 0).all()
    assert all((g[:, :, tk:] == 0).all() for g in grads[1:3]) and (grads[3][:, tk:] == 0).all()


def test_more_heads_than_stand_side_by_side():
    """a greatest length beyond every sequence leaves all tiles but the first ones empty and the heads in several groups: the same results"""
    lens, H = [70, 300, 129], 5
    q, k, v, c, do = _inputs(1, H, sum(lens), sum(lens), 128, 64, 128, HF, seed=6)
    cu = torch.tensor([0, 70, 370, 499], dtype=torch.int32, device=DEV)
    want, grads = _step(q, k, v, c, do, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=300, max_seqlen_k=300)
    out, more = _step(q, k, v, c, do, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=8192, max_seqlen_k=8192)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(more, grads))


@pytest.mark.parametrize('dtype', [HF, BF])
@pytest.mark.parametrize('E,R,Ev,causal', [(64, 32, 64, True), (128, 64, 128, True), (72, 64, 40, False)])
def test_many_workgroups(E, R, Ev, causal, dtype):
    """more tiles of queries than two for a CU, of which a few heads are looked at: rows with few keys, and past those whose delta comes from P"""
    B, H, Sq, Sk = 12, 24, 330, 333
    q, k, v, c, do = _inputs(B, H, Sq, Sk, E, R, Ev, dtype, seed=E)
    out, grads = _step(q, k, v, c, do, causal)
    for b, h in ((0, 0), (5, 23), (11, 7)):
        one = [t[b, h:h + 1] for t in (q, k, v)]
        alone, g1 = _step(*(t[None] for t in one), c[b:b + 1], do[b:b + 1, h:h + 1], causal)
        _check(*one, c[b], do[b, h:h + 1], causal, 1 / math.sqrt(E + R), out[b, h:h + 1], None, [grads[0][b, h:h + 1], grads[1][b, h:h + 1], grads[2][b, h:h + 1], g1[3][0]])
        assert_within('out', out[b, h:h + 1], alone[0], torch.zeros(()))


def test_offsets_outside_the_tensors():
    """what they name past the rows is not there, and neither are rows past the greatest length"""
    q, k, v, c, do = _inputs(1, 2, 200, 200, 64, 32, 64, BF, seed=4)
    cu = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    want, _ = _step(q, k, v, c, do, cu_seqlens_q=cu(0, 90, 200), cu_seqlens_k=cu(0, 90, 200), max_seqlen_q=110, max_seqlen_k=110)
    out, _ = _step(q, k, v, c, do, cu_seqlens_q=cu(-5, 90, 10 ** 9), cu_seqlens_k=cu(-9, 90, 2 ** 31 - 1), max_seqlen_q=110, max_seqlen_k=110)
    assert torch.equal(out, want)


@pytest.mark.parametrize('Sq,Sk', [(0, 0), (0, 5), (5, 0)])
def test_nothing_to_do(Sq, Sk):
    q, k, v, c, do = _inputs(1, 2, Sq, Sk, 64, 32, 64, BF)
    out, grads = _step(q, k, v, c, do)
    assert out.shape == (1, 2, Sq, 64) and (out == 0).all()
    for g, t in zip(grads, (q, k, v, c)):
        assert g.shape == t.shape and (g == 0).all()
    q, k, v, c, do = _inputs(0, 2, 30, 40, 64, 32, 64, BF)
    out, grads = _step(q, k, v, c, do)
    assert out.shape == (0, 2, 30, 64) and [g.shape for g in grads] == [t.shape for t in (q, k, v, c)]


def test_no_heads():
    q, k, v, c, do = _inputs(2, 0, 30, 40, 64, 32, 64, BF)
    out, grads = _step(q, k, v, c, do)
    assert out.shape == (2, 0, 30, 64) and [g.shape for g in grads] == [t.shape for t in (q, k, v, c)] and (grads[3] == 0).all()


@pytest.mark.parametrize('Sq', [1, 70, 128])
def test_rows_that_share_memory(Sq):
    """the gradient of a sum over rows, the same query for all of them, a single row whose stride says nothing: nothing of them lies behind the last row"""
    q, k, v, c, do = _inputs(2, 3, Sq, 100, 64, 32, 64, HF, seed=12)
    one = lambda t: t[:, :, :1].expand(-1, -1, Sq, -1)
    flat = lambda t: t.as_strided(t.shape, (t.stride(0), t.stride(1), 0, 1)) if Sq == 1 else one(t)
    for qq, dd in ((q, one(do)), (one(q), do), (flat(q), flat(do))):
        want, wgrads = _step(qq.contiguous(), k, v, c, dd.contiguous())
        out, grads = _step(qq, k, v, c, dd)
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, wgrads))


@pytest.mark.parametrize('scale', [0.0, -0.1, 3.0, 1e-3])
def test_scales(scale):
    q, k, v, c, do = _inputs(1, 2, 150, 150, 128, 64, 128, BF, seed=5)
    out, grads = _step(q, k, v, c, do, scale=scale)
    _check(q[0], k[0], v[0], c[0], do[0], True, scale, out[0], None, [g[0] for g in grads])


@pytest.mark.parametrize('order', [1, -1])
def test_the_largest_scores_come_first_or_last(order):
    """the running maximum moves at every tile, or never; scores far past the range of exp"""
    q, k, v, c, do = _inputs(1, 2, 300, 300, 64, 32, 64, BF, seed=6)
    size = torch.linspace(0.1, 30, 300, device=DEV)
    size = size if order > 0 else size.flip(0)
    k, c = (k * size[:, None]).to(BF), (c * size[:, None]).to(BF)
    out, grads = _step(q, k, v, c, do, scale=0.3)
    _check(q[0], k[0], v[0], c[0], do[0], True, 0.3, out[0], None, [g[0] for g in grads])


def test_strides_alignment_and_shared_storage():
    q, k, v, c, do = _inputs(2, 3, 130, 130, 64, 32, 64, HF, seed=7)
    want, wgrads = _step(q, k, v, c, do)
    odd = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t)             # an unaligned base
    wide = lambda t: torch.zeros(*t.shape[:-1], t.shape[-1] + 4, dtype=t.dtype, device=DEV)[..., 4:].copy_(t)     # rows no multiple of 16 bytes apart
    for f in (odd, wide, lambda t: t.contiguous()):
        out, grads = _step(f(q), f(k), f(v), f(c), f(do))
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, wgrads))
    # one key and value for all heads, seen through an expanded view
    k1, v1 = k[:, :1].expand(-1, 3, -1, -1), v[:, :1].expand(-1, 3, -1, -1)
    out, grads = _step(q, k1, v1, c, do)
    full, fgrads = _step(q, k1.contiguous(), v1.contiguous(), c, do)
    assert torch.equal(out, full) and all(torch.equal(a, b) for a, b in zip(grads, fgrads))


def test_gradient_of_a_broadcast_key():
    """leaves that the call sees expanded get the sum of their uses"""
    from aotriton_amd import torch_ops
    q, k, v, c, do = _inputs(2, 3, 90, 90, 64, 32, 64, BF, seed=8)
    c1 = c[:1].detach().requires_grad_(True)
    out = torch_ops.latent_attention(q, k, v, c1.expand(2, -1, -1))
    (got,) = torch.autograd.grad(out, c1, do)
    _, grads = _step(q, k, v, c[:1].expand(2, -1, -1), do)
    assert torch.equal(got, grads[3].sum(0, keepdim=True).to(BF))


def test_results_do_not_change_and_other_streams():
    x = _inputs(2, 5, 777, 777, 128, 64, 128, BF, seed=10)
    want = _step(*x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            got.append(_step(*x))
    torch.cuda.synchronize()
    for out, grads in got:
        assert torch.equal(out, want[0]) and all(torch.equal(a, b) for a, b in zip(grads, want[1]))


@pytest.mark.parametrize('packed', [False, True])
def test_captured_step(packed):
    """forward and backward in a graph, replayed on new values with eager work between the replays"""
    sets = [_inputs(1, 4, 400, 400, 64, 32, 64, HF, seed=20 + i) for i in range(3)]
    kw = {}
    if packed:
        cu = torch.tensor([0, 130, 390], dtype=torch.int32, device=DEV)
        kw = dict(cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=300, max_seqlen_k=300)
    static = [t.clone() for t in sets[0]]
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        _step(*static, **kw)
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = _step(*static, **kw)
    for values in sets + sets[:1]:
        for s, x in zip(static, values):
            s.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = _step(*values, **kw)
        assert torch.equal(out, want[0])
        assert all(torch.equal(a, b) for a, b in zip(grads, want[1]))


def test_compiled_and_traced():
    from aotriton_amd import torch_ops
    q, k, v, c, do = _inputs(1, 2, 100, 100, 64, 32, 64, BF, seed=11)
    args = (q, k, v, c, None, None, 0, 0, True, 0.125)
    torch.library.opcheck(torch.ops.aotriton_amd.latent_attention_forward, args, test_utils=('test_schema', 'test_faketensor'))
    out, lse = _raw(q, k, v, c, True, 0.125)
    torch.library.opcheck(torch.ops.aotriton_amd.latent_attention_backward, (do, q, k, v, c, out, lse) + args[4:],
                          test_utils=('test_schema', 'test_faketensor'))

    def step(q, k, v, c):
        return torch_ops.latent_attention(q, k, v, c).transpose(1, 2).flatten(2)
    torch._dynamo.reset()
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, c)]
    a, b = step(*leaves), torch.compile(step, backend='aot_eager', fullgraph=True)(*leaves)
    assert torch.equal(a, b)
    up = torch.randn_like(a)
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(a, leaves, up), torch.autograd.grad(b, leaves, up)))


def test_second_derivatives_are_refused():
    from aotriton_amd import torch_ops
    q, k, v, c, do = _inputs(1, 1, 20, 20, 64, 32, 64, BF)
    q = q.detach().requires_grad_(True)
    (dq,) = torch.autograd.grad(torch_ops.latent_attention(q, k, v, c), q, do, create_graph=True)
    with pytest.raises(RuntimeError, match='second derivatives'):
        dq.sum().backward()


def test_gradients_against_differences():
    """along a direction, in steps that the types' half steps leave visible: (f(x + h d) - f(x - h d)) / 2 h.  The outputs are rounded by a
    half step u each: the difference of the sums is off by u |out| |do| / h, and by h^2 / 6 times a third derivative, which for scores of
    this size is below the first"""
    from aotriton_amd import torch_ops
    x = _inputs(1, 2, 70, 70, 64, 32, 64, HF, seed=12)
    do = x[4].float()
    _, grads = _step(*x)
    f = lambda t: (torch_ops.latent_attention(*t).float() * do).sum().double()
    g = torch.Generator().manual_seed(13)
    for i in range(4):
        d = torch.randn(x[i].shape, generator=g).to(DEV)
        h = 2.0 ** -4
        up, down = (x[i].float() + h * d).half(), (x[i].float() - h * d).half()
        step = (up.float() - down.float()).double()          # what was added in fact
        a, b = (list(x[:4]) for _ in range(2))
        a[i], b[i] = up, down
        got = float(f(a) - f(b))
        want = float((grads[i].double() * step).sum())
        outs = torch_ops.latent_attention(*x[:4]).double()
        # (each of n outputs is rounded apart from the others: their sum by a few times the root of the sum of squares)
        off = 6 * 2.0 ** -11 * float((outs.abs() * do.double().abs()).norm()) + 0.02 * float((grads[i].double() * step).norm()) + 0.01 * abs(want)
        assert abs(got - want) < off, (i, got, want, off)


# ---- dQ with two waves on a SIMD: calls with more than two workgroups for a CU -----------------------------------------------

def _many(heads, tiles):
    """query tiles of 128 over all heads, which choose the kernel"""
    assert heads * tiles > 2 * torch.cuda.get_device_properties(0).multi_processor_count


def _offsets(lens, first=0):
    return torch.tensor([first + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)


@pytest.mark.parametrize('dtype', [HF, BF])
@pytest.mark.parametrize('E,R,Ev,causal,scale', [(128, 64, 128, True, None), (64, 32, 64, True, -0.1), (72, 64, 40, False, None), (128, 64, 128, False, 0.0), (128, 64, 128, True, 1.0)])
def test_packed_gradients_of_many_workgroups(E, R, Ev, causal, scale, dtype):
    """sequences without queries or keys, of one tile and of several, rows before the first key; the shared part's gradient over all heads"""
    lens_q, lens_k = [1, 300, 0, 77, 257, 5, 40, 64, 150], [1, 300, 7, 200, 257, 2, 0, 64, 90]
    H, tq, tk, pad = 64, sum(lens_q), sum(lens_k), 3
    _many(H, tq // 128 + (len(lens_q) + 1) // 2)
    q, _, _, _, do = _inputs(1, H, tq + pad, 1, E, R, Ev, dtype, seed=31)
    _, k, v, c, _ = _inputs(1, H, 1, tk + pad, E, R, Ev, dtype, seed=32)
    for t in (q, do):
        t[:, :, tq:] = float('nan')
    for t in (k, v):
        t[:, :, tk:] = float('inf')
    c[:, tk:] = float('nan')
    cq, ck = _offsets(lens_q), _offsets(lens_k)
    out, grads = _step(q, k, v, c, do, causal, scale, cu_seqlens_q=cq, cu_seqlens_k=ck, max_seqlen_q=max(lens_q), max_seqlen_k=max(lens_k))
    s = 1 / math.sqrt(E + R) if scale is None else scale
    for i in range(len(lens_q)):
        a, b = slice(int(cq[i]), int(cq[i + 1])), slice(int(ck[i]), int(ck[i + 1]))
        _check(q[0][:, a], k[0][:, b], v[0][:, b], c[0][b], do[0][:, a], causal, s, out[0][:, a], None,
               [grads[0][0][:, a], grads[1][0][:, b], grads[2][0][:, b], grads[3][0][b]], f'sequence {i} ')
    assert (grads[0][:, :, tq:] == 0).all() and all((g[:, :, tk:] == 0).all() for g in grads[1:3]) and (grads[3][:, tk:] == 0).all()


@pytest.mark.parametrize('dtype', [HF, BF])
@pytest.mark.parametrize('B,H,Sq,Sk,E,R,Ev,causal,scale', [
    (12, 48, 40, 40, 128, 64, 128, True, None),        # one tile of keys: what dS loses in 16 bits goes through the product as well
    (18, 30, 100, 64, 64, 32, 64, False, -0.2),
    (9, 64, 90, 30, 64, 64, 64, True, None),           # queries before the first key
    (5, 60, 140, 100, 128, 40, 72, True, 0.0),
    (6, 50, 200, 290, 128, 64, 128, True, 2.0)])       # delta from O
def test_gradients_of_many_workgroups(B, H, Sq, Sk, E, R, Ev, causal, scale, dtype):
    """every head of a few batches, and with them the shared part's gradient"""
    _many(B * H, (Sq + 127) // 128)
    q, k, v, c, do = _inputs(B, H, Sq, Sk, E, R, Ev, dtype, seed=Sq + 1)
    out, grads = _step(q, k, v, c, do, causal, scale)
    for b in (0, B - 1):
        _check(q[b], k[b], v[b], c[b], do[b], causal, 1 / math.sqrt(E + R) if scale is None else scale, out[b], None, [g[b] for g in grads], f'sequence {b} ')


@pytest.mark.parametrize('Sq,Sk', [(70, 100), (1, 60), (128, 300)])
def test_rows_that_share_memory_of_many_workgroups(Sq, Sk):
    B, H = 11, 50
    _many(B * H, 1)
    q, k, v, c, do = _inputs(B, H, Sq, Sk, 64, 32, 64, HF, seed=33)
    one = lambda t: t[:, :, :1].expand(-1, -1, t.shape[2], -1)
    heads = lambda t: t[:, :1].expand(-1, H, -1, -1)
    for qq, kk, vv, dd in ((q, k, v, one(do)), (one(q), k, v, do), (q, heads(k), heads(v), one(do))):
        want, wgrads = _step(qq.contiguous(), kk.contiguous(), vv.contiguous(), c, dd.contiguous())
        out, grads = _step(qq, kk, vv, c, dd)
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, wgrads))
    _check(q[3], k[3], v[3], c[3], do[3, :, :1].expand(-1, Sq, -1), True, 1 / math.sqrt(96), *(lambda o, g: (o[3], None, [x[3] for x in g]))(*_step(q, k, v, c, one(do))))


# ---- packed sequences whose keys are cut into parts -----------------------------------------------------------------------------

@pytest.mark.parametrize('dtype', [HF, BF])
@pytest.mark.parametrize('E,R,Ev,causal,top', [(128, 64, 128, True, 2100), (64, 32, 64, False, 2100), (40, 8, 24, True, 9000)])
def test_packed_keys_cut_into_parts(E, R, Ev, causal, top, dtype):
    """few rows, long and short keys, none; a greatest length beyond them all cuts the keys more finely"""
    lens_q, lens_k, H, pad = [130, 1, 0, 64, 7, 33], [2100, 1500, 40, 0, 1030, 3], 2, 5
    tq, tk = sum(lens_q), sum(lens_k)
    q, _, _, _, do = _inputs(1, H, tq + pad, 1, E, R, Ev, dtype, seed=41)
    _, k, v, c, _ = _inputs(1, H, 1, tk + pad, E, R, Ev, dtype, seed=42)
    q[:, :, tq:] = float('nan')
    k[:, :, tk:] = float('inf')
    cq, ck = _offsets(lens_q), _offsets(lens_k)
    scale = 0.1
    out, lse = torch.ops.aotriton_amd.latent_attention_forward(q, k, v, c, cq, ck, max(lens_q), top, causal, scale)
    for i in range(len(lens_q)):
        a, b = slice(int(cq[i]), int(cq[i + 1])), slice(int(ck[i]), int(ck[i + 1]))
        _check(q[0][:, a], k[0][:, b], v[0][:, b], c[0][b], do[0][:, a], causal, scale, out[0][:, a], lse[:, a], None, f'sequence {i} ')
    assert (out[:, :, tq:] == 0).all()


def test_scratch_of_a_ragged_batch():
    """one long sequence and many short ones: scratch goes by the rows, a slab of 32 of them and two words a row for every part (16 at most), and no
    sequence has more than one slab that is not full"""
    lens, E = [2048] + [4] * 199, 128
    q, k, v, c, do = _inputs(1, 1, sum(lens), sum(lens), E, 64, E, BF, seed=43)
    cu = _offsets(lens)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out, lse = torch.ops.aotriton_amd.latent_attention_forward(q, k, v, c, cu, cu, 2048, 2048, True, 0.05)
    used = torch.cuda.max_memory_allocated() - before
    slabs = sum(lens) // 32 + len(lens)
    assert used <= out.numel() * 2 + lse.numel() * 4 + 16 * slabs * (32 * E * 4 + 256) + (8 << 20)
    for i in (0, 1, 100, 199):
        a = slice(int(cu[i]), int(cu[i + 1]))
        _check(q[0][:, a], k[0][:, a], v[0][:, a], c[0][a], do[0][:, a], True, 0.05, out[0][:, a], lse[:, a], None, f'sequence {i} ')


# ---- rows of no sequence ------------------------------------------------------------------------------------------------------

def _poison():
    """memory that the next calls are given holds NaN"""
    made = [torch.full((n,), float('nan'), device=DEV) for n in (1 << 12, 1 << 16, 1 << 18, 1 << 20, 1 << 22) for _ in range(6)]
    torch.cuda.synchronize()
    del made


@pytest.mark.parametrize('dtype', [HF, BF])
@pytest.mark.parametrize('H', [3, 80])
@pytest.mark.parametrize('causal', [True, False])
def test_rows_in_front_and_past_the_greatest_length(causal, H, dtype):
    """offsets that do not begin at 0, sequences longer than the greatest length: what no sequence has is not there, may hold anything, and gets zeros"""
    cu_q, cu_k, top_q, top_k, E, R, Ev = [5, 60, 60, 200, 203], [9, 80, 100, 250, 251], 100, 120, 64, 32, 64
    q, _, _, _, do = _inputs(1, H, 230, 1, E, R, Ev, dtype, seed=51)
    _, k, v, c, _ = _inputs(1, H, 1, 260, E, R, Ev, dtype, seed=52)
    has = lambda cu, top: [slice(cu[i], cu[i] + min(cu[i + 1] - cu[i], top)) for i in range(len(cu) - 1)]
    rows_q, rows_k = has(cu_q, top_q), has(cu_k, top_k)
    off = lambda n, rows: torch.tensor([not any(r.start <= i < r.stop for r in rows) for i in range(n)], device=DEV)
    off_q, off_k = off(230, rows_q), off(260, rows_k)
    for t in (q, do):
        t[:, :, off_q] = float('nan')
    for t in (k, v):
        t[:, :, off_k] = float('inf')
    c[:, off_k] = float('nan')
    cu = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    _poison()
    out, grads = _step(q, k, v, c, do, causal, cu_seqlens_q=cu(cu_q), cu_seqlens_k=cu(cu_k), max_seqlen_q=top_q, max_seqlen_k=top_k)
    for i, (a, b) in enumerate(zip(rows_q, rows_k)):
        _check(q[0][:, a], k[0][:, b], v[0][:, b], c[0][b], do[0][:, a], causal, 1 / math.sqrt(E + R), out[0][:, a], None,
               [grads[0][0][:, a], grads[1][0][:, b], grads[2][0][:, b], grads[3][0][b]], f'sequence {i} ')
    assert (out[:, :, off_q] == 0).all() and (grads[0][:, :, off_q] == 0).all()
    assert all((g[:, :, off_k] == 0).all() for g in grads[1:3]) and (grads[3][:, off_k] == 0).all()


@pytest.mark.parametrize('top_q,top_k', [(0, 0), (0, 9), (9, 0)])
def test_greatest_lengths_of_nothing(top_q, top_k):
    q, k, v, c, do = _inputs(1, 2, 40, 50, 64, 32, 64, BF, seed=53)
    cu = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    _poison()
    out, grads = _step(q, k, v, c, do, cu_seqlens_q=cu(0, 30, 40), cu_seqlens_k=cu(0, 20, 50), max_seqlen_q=top_q, max_seqlen_k=top_k)
    assert all((t == 0).all() for t in (out, *grads))


def test_offsets_that_end_outside_or_descend():
    """in front of the tensors, behind them, falling: inside the tensors whatever comes of it, and rows that a sequence has are right"""
    q, k, v, c, do = _inputs(1, 2, 200, 200, 64, 32, 64, BF, seed=54)
    cu = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    want, wgrads = _step(q, k, v, c, do, cu_seqlens_q=cu(0, 90, 200), cu_seqlens_k=cu(0, 90, 200), max_seqlen_q=110, max_seqlen_k=110)
    out, grads = _step(q, k, v, c, do, cu_seqlens_q=cu(-5, 90, 10 ** 9), cu_seqlens_k=cu(-9, 90, 2 ** 31 - 1), max_seqlen_q=110, max_seqlen_k=110)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, wgrads))
    out, grads = _step(q, k, v, c, do, cu_seqlens_q=cu(300, 250), cu_seqlens_k=cu(300, 250), max_seqlen_q=110, max_seqlen_k=110)
    assert all((t == 0).all() for t in (out, *grads))
    for odd in (cu(150, 90, 200), cu(10 ** 9, -5, 2 ** 31 - 1, -2 ** 31)):
        _step(q, k, v, c, do, cu_seqlens_q=odd, cu_seqlens_k=odd, max_seqlen_q=110, max_seqlen_k=110)


def test_captured_rows_of_no_sequence():
    """offsets that change between the replays of a graph"""
    cu = torch.tensor([0, 60, 200], dtype=torch.int32, device=DEV)
    x = _inputs(1, 3, 230, 230, 64, 32, 64, HF, seed=55)
    kw = dict(cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=100, max_seqlen_k=100)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        _step(*x, **kw)
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = _step(*x, **kw)
    for offsets in ([0, 60, 200], [7, 60, 90], [0, 0, 230], [100, 230, 230], [0, 60, 200]):
        cu.copy_(torch.tensor(offsets, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = _step(*x, **kw)
        assert torch.equal(out, want[0]) and all(torch.equal(a, b) for a, b in zip(grads, want[1]))
        covered = torch.zeros(230, dtype=torch.bool, device=DEV)
        for a, b in zip(offsets, offsets[1:]):
            covered[a:min(b, a + 100)] = True
        assert (out[:, :, ~covered] == 0).all() and all((g[:, :, ~covered] == 0).all() for g in grads[:3]) and (grads[3][:, ~covered] == 0).all()
