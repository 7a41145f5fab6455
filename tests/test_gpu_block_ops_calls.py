"""Calls of the operators around a block's projections that the tests of each
operator do not make."""
import pytest
import torch
from torch.autograd import forward_ad

from block_refs import assert_close, linear_w4 as exact_w4
from w8a8 import axial_rope, block_norm, kernels, linear_w4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('rows,sections,far', [(20011, (64,), 64), (5003, (24, 20, 20), 1000), (4001, (16, 16, 16), 300000)])
def test_sine_and_cosine_keep_their_bits(gpu, rows, sections, far):
    """Each is within 1.3 * 2^-24 (u = 2^-24): the rest |x| <= pi / 4 is rounded once
    (0.5 u, times the other function, at most 0.88 and 0.71), the last sum once (0.5
    u), the terms before it add 0.25 u (sine) and 0.25 u + 0.16 u (cosine), the series'
    ends 0.03 u: 1.22 u and 1.28 u. The fp64 angle is within 2^-50 of its size."""
    g = torch.Generator().manual_seed(rows)
    pos = (torch.rand((rows, len(sections)), generator=g) * far).to(gpu)
    inv, axis = axial_rope.ladder(sections, device=gpu)
    f = axial_rope.freqs(pos, inv, axis, dtype=torch.float32)[0, :, 0].double()
    phi = pos.double()[:, axis.long()] * inv
    bound = 1.3 * 2.0 ** -24 + 2.0 ** -50 * phi.abs()
    for got, exact in ((f[..., 0, 0], phi.cos()), (f[..., 1, 0], phi.sin()), (f[..., 0, 1], -phi.sin()),
                       (f[..., 1, 1], phi.cos())):
        assert bool(((got - exact).abs() <= bound).all()), float((got - exact).abs().max())


@pytest.mark.parametrize('m', [1, 8, 30, 64, 130])
@pytest.mark.parametrize('group,zeros', [(32, False), (64, True), (128, True)])
def test_subnormal_scales(gpu, m, group, zeros):
    """FP16 scales below 2^-14, as small weights have them, keep their value."""
    g = torch.Generator().manual_seed(m)
    n, k = 72, 384
    codes = torch.randint(0, 16, (n, k), generator=g)
    scales = (torch.randint(1, 1024, (k // group, n), generator=g).float() * 2.0 ** -24).half()
    assert float(scales.max()) < 2.0 ** -14 and float(scales.min()) > 0
    z = torch.randint(0, 16, (k // group, n), generator=g).to(torch.uint8) if zeros else None
    x = (torch.randn((m, k), generator=g) * 300).half()
    args = [t.to(gpu) if t is not None else None for t in (x, codes, scales, z)]
    y = linear_w4.linear(args[0], linear_w4.pack(args[1]), args[2], args[3])
    assert_close(y, *exact_w4(*args), 'outputs')
    w = (torch.randn((n, k), generator=g) * 0.02).to(gpu)
    mod = linear_w4.LinearW4(k, n, group_size=group, zeros=zeros, device=gpu).load_weight(w / 512)
    assert float(mod.scales.max()) < 2.0 ** -14
    y = mod(args[0])
    assert_close(y, *exact_w4(args[0], linear_w4.unpack(mod.codes), mod.scales, mod.zeros), 'module')


def test_forward_mode_tangents_are_refused(gpu):
    x = torch.zeros((2, 256), dtype=torch.float16, device=gpu)
    q = torch.zeros((2, 4, 128), dtype=torch.float16, device=gpu)
    inv, axis = axial_rope.ladder((16, 16, 16), device=gpu)
    pos = torch.zeros((2, 3), device=gpu)
    codes = torch.zeros((16, 32), dtype=torch.int32, device=gpu)
    scales = torch.ones((2, 16), dtype=torch.float16, device=gpu)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: block_norm.residual_norm(dual(x), x, eps=1e-6),
                     lambda: block_norm.residual_norm(x, x, eps=1e-6, weight=dual(torch.ones(256, device=gpu))),
                     lambda: block_norm.residual_norm(x, x, out=dual(x)),
                     lambda: axial_rope.rotate(dual(q), None, pos, inv, axis),
                     lambda: axial_rope.freqs(dual(pos), inv, axis),
                     lambda: linear_w4.linear(dual(x), codes, scales),
                     lambda: linear_w4.linear(x, codes, scales, bias=dual(scales[0]))):
            with pytest.raises(ValueError, match='no gradient'):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match='no gradient'):
                call()
        block_norm.residual_norm(x, x, eps=1e-6)


@pytest.mark.parametrize('out', [False, True])
def test_residuals_of_other_rows_are_refused(gpu, out):
    """A residual has x's leading sizes, or its rows in one dimension."""
    x = torch.randn((2, 3, 256), device=gpu).half()
    codes, scales, _ = linear_w4.quantize_weight(torch.randn((16, 256)))
    codes, scales = codes.to(gpu), scales.to(gpu)
    r = torch.randn((2, 3, 16), device=gpu).half()
    kw = dict(out=torch.zeros((6, 16), dtype=torch.float16, device=gpu)) if out else {}
    want = linear_w4.linear(x, codes, scales, residual=r)
    assert torch.equal(linear_w4.linear(x, codes, scales, residual=r.view(6, 16), **kw).view(2, 3, 16), want)
    assert torch.equal(linear_w4.linear(x, codes, scales, residual=r, **kw).view(2, 3, 16), want)
    assert torch.equal(linear_w4.linear(x[0, 0], codes, scales, residual=r[0, :1]), want[0, 0])
    for same in (r.view(6, 1, 16), r.view(1, 2, 3, 16)):
        assert torch.equal(linear_w4.linear(x, codes, scales, residual=same, **kw).view(2, 3, 16), want)
    assert torch.equal(linear_w4.linear(x.view(6, 256), codes, scales, residual=r, **kw).view(2, 3, 16), want)
    for bad in (r.transpose(0, 1).contiguous(), r[:1], r[..., :8], r.view(2, 3, 8, 2)):
        with pytest.raises(ValueError, match='residual'):
            linear_w4.linear(x, codes, scales, residual=bad, **kw)


@pytest.mark.parametrize('heads_first', [False, True])
@pytest.mark.parametrize('rows,heads,dim', [(37, 5, 128), (1, 3, 64), (9, 1, 96)])
def test_interleaved_heads_in_place(gpu, rows, heads, dim, heads_first):
    """q and k of a buffer [rows, heads, 3, dim] (or [heads, 3, rows, dim]) turn in
    place: their heads lie between each other and share nothing."""
    g = torch.Generator().manual_seed(rows)
    shape = (heads, 3, rows, dim) if heads_first else (rows, heads, 3, dim)
    buf = torch.randn(shape, generator=g).half().to(gpu)

    def views(t):
        return tuple(t[:, i].transpose(0, 1) if heads_first else t[:, :, i] for i in range(3))
    pos = torch.randint(0, 500, (rows, 2), generator=g).to(gpu)
    inv, axis = axial_rope.ladder((dim // 4, dim // 4), device=gpu)
    q, k, v = views(buf)
    keep = v.clone()
    want = axial_rope.rotate(q.contiguous(), k.contiguous(), pos, inv, axis)
    got = axial_rope.rotate(q, k, pos, inv, axis, out=(q, k))
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, keep)


def test_writes_into_given_outputs_are_counted(gpu):
    """A tensor that autograd has saved elsewhere and that a call writes into is not
    taken for unchanged by a later backward pass."""
    h = torch.randn((4, 256), device=gpu).half()
    q = torch.randn((4, 2, 64), device=gpu).half()
    inv, axis = axial_rope.ladder((32,), device=gpu)
    pos = torch.zeros((4, 1), dtype=torch.int64, device=gpu)
    codes, scales, _ = linear_w4.quantize_weight(torch.randn((256, 256)))
    codes, scales = codes.to(gpu), scales.to(gpu)
    signs = torch.zeros(256, dtype=torch.int32, device=gpu)
    for call in (lambda t: block_norm.residual_norm(t, h, out=t),
                 lambda t: block_norm.residual_norm(t, h, eps=1e-6, quantize=True, signs=signs, out=t),
                 lambda t: linear_w4.linear(h, codes, scales, residual=t, out=t)):
        x = torch.randn((4, 256), device=gpu).half()
        weight = torch.ones(256, dtype=torch.float16, device=gpu, requires_grad=True)
        y = (x * weight).sum()                                  # saves x
        before = x._version
        call(x)
        assert x._version > before
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            y.backward()
    for turn in (axial_rope.rotate, kernels.axial_rope):
        before = q._version, (k := q.clone())._version
        turn(q, k, pos, inv, axis, out=(q, k))
        assert q._version > before[0] and k._version > before[1]
    with torch.inference_mode():
        t = torch.zeros((4, 256), dtype=torch.float16, device=gpu)
    block_norm.residual_norm(t, h, out=t)                       # a tensor without a count
    with torch.inference_mode():
        block_norm.residual_norm(t, h, out=t)
        kernels.residual_norm(t, h, out=t)
