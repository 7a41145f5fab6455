"""Attention in 64 bits and what its 16-bit form may differ by.

The kernels hold scores, maxima, sums and products in fp32 and round twice to
the operands' type T (half a step, u = eps / 2 relative): p, relative to the
running maximum, before its product with v, and the output. With
A = sum p |v| / sum p:
  * p's rounding:            u (A + |o|) if the sum in the denominator takes
                             the rounded p, as with 16-bit values
                             (sum of p d_j (v_j - o) / sum p with |d_j| <= u),
                             u A if it does not; in fp16 what lies below 2^-24 is lost, by
                             half of that at most: 2^-25 sum |v| / sum p,
                             where sum p >= 1 relative to the maximum
  * the score's sum of D products and its scaling: (D + 4) 2^-24 of the sum of
    magnitudes, |c| sum |q k|, and exp2 within 2^-22, so p is off by d relative;
    numerator and denominator: 2 d A
  * the sums over n keys, and their rescaling at most once a block of 32:
    (n + n / 32 + 8) 2^-24 A, twice
  * the output:              u |o| (in fp16 2^-25 where it is subnormal)
A cache of codes adds two fp32 products before p's rounding (in (n + 8)
above). Codes are multiplied as fp16 whatever T is, so that p's fp16 loss counts
for both, relative to the largest scale of v: 2^-25 sum max(s) |code|; and q of
bf16, scaled by a power of 2 to a largest from 1 to 2, loses 2^-25 of that at
most in a small element: d has |c| D 2^-25 2 max|q| max|k| more.
"""
import math

import torch


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def attention64(q, k, v, scale, first=None, codes_scale=None):
    """(o, bound) of one head: q [nq, d], k, v [nk, d] in 64 bits; query i sees
    the keys before first[i] (all by default). o is 0 where there are none."""
    nq, nk = q.shape[0], k.shape[0]
    if nk == 0:
        z = torch.zeros((nq, v.shape[1]), dtype=torch.float64, device=q.device)
        return z, z
    t = (q @ k.t()) * scale
    seen = torch.ones((nq, nk), dtype=torch.bool, device=q.device)
    if first is not None:
        seen = torch.arange(nk, device=q.device)[None] < first[:, None]
    t = torch.where(seen, t, torch.full_like(t, -math.inf))
    top = t.amax(1, keepdim=True)
    p = torch.where(seen, torch.exp(t - torch.where(top == -math.inf, torch.zeros_like(top), top)), torch.zeros_like(t))
    total = p.sum(1, keepdim=True).clamp_min(1e-300)
    o = (p @ v) / total
    a = (p @ v.abs()) / total
    lost = torch.where(seen, 1.0, 0.0).double() @ (v.abs() if codes_scale is None else codes_scale)
    d = (q.shape[1] + 4) * 2.0 ** -24 * ((q.abs() @ k.abs().t()) * scale * seen).amax(1, keepdim=True) + 2.0 ** -22
    if codes_scale is not None:
        d = d + scale * q.shape[1] * 2.0 ** -24 * q.abs().amax(1, keepdim=True) * k.abs().max()
    return o, (a, lost, d, nk, codes_scale is not None)


def bound(o, parts, dtype):
    """The largest difference that attention64's comment allows."""
    if not isinstance(parts, tuple):
        return torch.zeros_like(o)
    a, lost, d, nk, codes = parts
    u = _u(dtype)
    tol = 2 * u * o.abs() + a * (u + 2 * d + 2 * (nk + nk / 32 + 8) * 2.0 ** -24)
    if dtype == torch.float16 or codes:
        tol = tol + 2.0 ** -25 * lost
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    return tol * 1.01 + 1e-37   # (the bound's own products of small terms)


def check(got, want, tol, what=''):
    got = got.double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (
        f'{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol).max()):.3g} of the '
        f'tolerance, first at {bad.nonzero()[0].tolist()}: {float(got[bad][0]):.6g} for {float(want[bad][0]):.6g}')


def check_packed(got, q, k, v, starts, k_starts, causal, scale, what=''):
    """got [rows, heads, dim] against 64 bits; rows behind the last sequence are not looked at."""
    group = q.shape[1] // k.shape[1]
    for b in range(len(starts) - 1):
        q0, q1, k0, k1 = starts[b], starts[b + 1], k_starts[b], k_starts[b + 1]
        nq, nk = q1 - q0, k1 - k0
        if nq == 0:
            continue
        first = torch.arange(nq, device=q.device) + nk - nq + 1 if causal else None
        for h in range(q.shape[1]):
            o, parts = attention64(q[q0:q1, h].double(), k[k0:k1, h // group].double(), v[k0:k1, h // group].double(),
                                   scale, first)
            check(got[q0:q1, h], o, bound(o, parts, q.dtype), f'{what} sequence {b} head {h}')


def quantize64(x):
    """(codes, fp32 scale) of the last dimension, by the row quantizer's definition."""
    f = x.float()
    scale = (f.abs().amax(-1) * torch.tensor(1.0 / 127.0, dtype=torch.float32, device=x.device)).clamp_min(1e-30)
    return (f / scale[..., None]).round().clamp(-128, 127).to(torch.int8), scale


def starts_of(lengths, device=None):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at, torch.tensor(at, dtype=torch.int32, device=device)


def table_of(lengths, page, gen, device, extra=2, width=None):
    """A page table of shuffled pages for sequences of these lengths, and the pages of its cache."""
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=gen)
    table = torch.full((len(lengths), width or max(max(need, default=0), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to(device), pages
