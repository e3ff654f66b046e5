"""Bounds on the errors of the operators for long contexts, from the roundings that they make, computed in 64 bits.

A rounding to the tensors' type is off by at most u = eps / 2 of the value (fp16 below 2^-14: by 2^-25).  The kernels keep scores,
probabilities, row sums, dP and dS in fp32 (sums of products of 16-bit numbers: off by at most (D + 8) 2^-24 of the sum of their absolute
values) and round
  P before O += P V and dV += P^T dO, dS before dQ += dS K and dK += dS^T Q, and each result at the end.
With e = what the scores are off by (twice: numerator and row sum; and 2^-20 for exp2 and the sums), P is off by a share u + 2 e."""
import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """What a rounding to the type, or a probability, is off by however small it is: half of fp16's least step 2^-24; for bf16, whose range is
    fp32's, the smallest normal number 2^-126, below which the exponential of the hardware (and a bf16 result) is 0."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def score_error(q, k, scale):
    """The most that a score (in units of exp) can be off by, over all of them."""
    d = q.shape[-1]
    if q.numel() == 0 or k.numel() == 0:
        return 0.0
    biggest = q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max() * abs(scale)
    return float((d + 8) * 2.0 ** -24 * biggest + 2.0 ** -20)


def out_bound(dtype, out, size, values, e):
    """size: sum of P |V|; values: sum of |V| over what may be seen."""
    u = half_step(dtype)
    return u * out.abs() + (1.01 * u + 2 * e) * size + smallest(dtype) * (values + 1) + 1e-30


def lse_bound(lse, e):
    return e + 2.0 ** -22 * (1 + lse.abs())


def grad_bounds(dtype, q, k, v, dout, seen, scale, out, size, p):
    """Elementwise bounds for dQ, dK, dV of one sequence (q (Hq, n, D), k (Hk, m, D)); p the probabilities."""
    u, tiny, e = half_step(dtype), smallest(dtype), score_error(q, k, scale)
    hk, g = k.shape[0], q.shape[0] // k.shape[0]
    kx, vx = (t.double().repeat_interleave(g, 0) for t in (k, v))
    qd, do = q.double(), dout.double()
    delta = (do * out).sum(-1, keepdim=True)
    dp = torch.matmul(do, vx.transpose(1, 2))
    ds = (p * (dp - delta)).abs()
    f32 = (q.shape[-1] + 8) * 2.0 ** -24
    # delta comes from the rounded output; dP and delta are sums in fp32
    o_off = out_bound(dtype, out, size, vx.abs().sum(1, keepdim=True), e)
    dp_off = f32 * torch.matmul(do.abs(), vx.abs().transpose(1, 2)) + (do.abs() * (o_off + f32 * out.abs())).sum(-1, keepdim=True)
    off = torch.where(seen, (1.01 * u + 2 * e) * ds + 1.01 * p * dp_off + tiny, 0.0)
    p_off = torch.where(seen, (1.01 * u + 2 * e) * p + tiny, 0.0)
    sums = 2.0 ** -24 * (g * q.shape[1] + k.shape[1] + 8)      # the long sums' own roundings, as a share of their absolute terms
    merge = lambda t: t.view(hk, g, *t.shape[1:]).sum(1)
    dq = torch.matmul(off + sums * ds, kx.abs()) * abs(scale)
    dk = merge(torch.matmul((off + sums * ds).transpose(1, 2), qd.abs())) * abs(scale)
    dv = merge(torch.matmul((p_off + sums * p).transpose(1, 2), do.abs()))
    return dq, dk, dv, u, tiny


def assert_within(name, got, want, bound):
    got, want = got.double().cpu(), want.double().cpu()
    bound = bound.double().cpu().expand_as(want)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert not torch.isnan(got).any(), f'{name}: NaN'
    same = got == want                        # (infinities)
    off = torch.where(same, 0.0, (got - want).abs() - bound)
    if off.numel() and off.max() > 0:
        at = off.argmax().item()
        raise AssertionError(f'{name}: {got.flatten()[at]:.6g} for {want.flatten()[at]:.6g}, allowed off by {bound.flatten()[at]:.3g}; '
                             f'{int((off > 0).sum())} of {off.numel()} values')
