"""64-bit statements of the operators around a block's projections, and the
tolerances of their outputs."""
import torch


def half_step(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def subnormal_step(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def assert_close(got, exact, slack, what=''):
    """|got - exact| <= half a step of got's type at exact + slack (a tensor of
    absolute fp32 errors), and the same non-finite values."""
    got64, dt = got.double().cpu(), got.dtype
    exact, slack = exact.double().cpu(), slack.double().cpu()
    fine = torch.isfinite(exact)
    assert torch.equal(torch.isnan(got64), torch.isnan(exact)), what
    assert torch.equal(got64[~fine & ~torch.isnan(exact)], exact[~fine & ~torch.isnan(exact)]), what
    bound = exact.abs() * half_step(dt) + slack * (1 + half_step(dt)) + subnormal_step(dt)
    bad = fine & ~((got64 - exact).abs() <= bound)
    if bad.any():
        i = tuple(torch.nonzero(bad)[0].tolist())
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.numel()} too far; first {i}: got {got64[i]}, exact '
                             f'{exact[i]}, allowed {bound[i]}')


def residual_update(x, branch, *, post_weight=None, post_eps=None, gate=None, labels=None, residual_scale=1.0,
                    branch_scale=1.0):
    """(x' before its rounding, absolute fp32 slack)."""
    b = branch.double()
    if post_eps is not None:
        b = b / (b.square().mean(-1, keepdim=True) + post_eps).sqrt()
        if post_weight is not None:
            b = b * post_weight.double()
    u = b * branch_scale
    if gate is not None:
        u = u * gate.double()[labels.long().clamp(0, gate.shape[0] - 1)]
    r = x.double() * residual_scale
    # The norm's sum of squares adds 16 terms, 6 butterfly steps and at most 512
    # unit sums, all positive: relative 2^-24 each, halved by the root (under
    # 2^-15 for the widest rows here, 2^-18 for 6 unit sums); a dozen more
    # roundings follow.
    units = -(-x.shape[-1] // 1024)
    slack = (32 + units + 12) * 2.0 ** -24 * (u.abs() + r.abs())
    return r + u, slack


def rope(x, positions, inv_freq, axis, *, adjacent=False, gain=None, eps=1e-6):
    """(turned x, absolute fp32 slack) of x [rows, heads, dim]."""
    v = x.double()
    dim = v.shape[-1]
    if gain is not None:
        v = v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()
    n = inv_freq.numel()
    phi = positions.double()[:, axis.long().clamp(0, positions.shape[1] - 1)] * inv_freq.double()
    cos, sin = phi.cos()[:, None], phi.sin()[:, None]
    if adjacent:
        a, b = v[..., 0:2 * n:2], v[..., 1:2 * n:2]
    else:
        a, b = v[..., :n], v[..., n:2 * n]
    ra, rb = a * cos - b * sin, b * cos + a * sin
    out, size = v.clone(), v.abs().clone()
    both = a.abs() + b.abs()
    if adjacent:
        out[..., 0:2 * n:2], out[..., 1:2 * n:2] = ra, rb
        size[..., 0:2 * n:2] = size[..., 1:2 * n:2] = both
    else:
        out[..., :n], out[..., n:2 * n] = ra, rb
        size[..., :n] = size[..., n:2 * n] = both
    # Without a norm a channel that does not turn is copied. The norm's sum has
    # at most dim positive terms (2^-24 each, halved by the root), five more
    # roundings; sine and cosine are within 2^-22 (their series, the fraction's
    # rounding to fp32 times 2 pi) and two products and a sum follow.
    slack = size * ((dim / 2 + 5) * 2.0 ** -24 if gain is not None else 0.0)
    turned = torch.zeros(dim, dtype=torch.float64, device=x.device)
    turned[:2 * n] = 1
    return out, slack + size * turned * (2.0 ** -21 + 4 * 2.0 ** -24)


def linear_w4(x, codes, scales, zeros=None, *, bias=None, residual=None, gated=False):
    """(y before its rounding, absolute fp32 slack); codes [N, K] as integers."""
    n, k = codes.shape
    groups = scales.shape[0]
    group = k // groups
    z = torch.full_like(scales, 8.0, dtype=torch.float64) if zeros is None else zeros.double()
    s = scales.double()
    w = ((codes.double().reshape(n, groups, group) - z.t()[:, :, None]) * s.t()[:, :, None]).reshape(n, k)
    y = x.double() @ w.t()
    # Blocks of at most 128 inputs: sums of (16 + c) x and of x with at most 128
    # roundings each (2^-24 of their largest partial sum, at most the sum of
    # sizes), (16 + z) times the second taken off; then at most one addition a
    # block and one a wave (8) or k range (16).
    block = min(group, 128)
    size = x.double().abs().reshape(-1, groups, group).sum(-1) @ (s * (31.0 + 31.0))   # [M, N]
    slack = size * 2.0 ** -24 * (block + 4 + k // block + 24)
    if bias is not None:
        y = y + bias.double()
        slack = slack + y.abs() * 2.0 ** -24
    if gated:
        g, u = y.chunk(2, -1)
        sg, su = slack.chunk(2, -1)
        # d/dg silu is below 1.1; exp, the division and two products are each within 2^-22.
        y = g * torch.sigmoid(g) * u
        slack = 1.1 * sg * u.abs() + (g * torch.sigmoid(g)).abs() * su + 1.1 * sg * su + y.abs() * 2.0 ** -20
    if residual is not None:
        y = y + residual.double()
        slack = slack + y.abs() * 2.0 ** -24
    return y, slack
