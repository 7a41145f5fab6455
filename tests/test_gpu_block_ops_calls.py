"""Calls of the operators around a block's projections that the tests of each
operator do not make."""
import pytest
import torch

from w8a8 import axial_rope

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
