"""Calls of the operators around a block's projections without a GPU: refusals
and the 4-bit quantizer's range."""
import pytest
import torch

from w8a8 import linear_w4


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('symmetric', [True, False])
@pytest.mark.parametrize('size', [0.05, 0.02 / 512, 2.0 ** -18, 2.0 ** -22])
def test_small_weights_keep_their_steps(dtype, symmetric, size):
    """Scales may lie below the type's smallest normal (fp16: 2^-14), as those of
    weights that carry a residual divisor do. The ideal step is the range over the
    codes; its scale is half a unit in the last place off, or below the smallest
    normal at most one spacing more (never less: no weight is cut off). A weight is
    half a step off, and at the range's ends by what 15 steps lose with the scale."""
    g = torch.Generator().manual_seed(4)
    w = torch.randn((24, 256), generator=g) * size
    w[5, :64] = 0
    codes, scales, zeros = linear_w4.quantize_weight(w, 64, symmetric=symmetric, dtype=dtype)
    back = linear_w4.dequantize_weight(codes, scales, zeros).double().reshape(24, 4, 64)
    groups = w.double().reshape(24, 4, 64)
    if symmetric:
        ideal = groups.abs().amax(-1, keepdim=True) / 7
    else:
        ideal = (groups.amax(-1, keepdim=True).clamp_min(0) - groups.amin(-1, keepdim=True).clamp_max(0)) / 15
    info = torch.finfo(dtype)
    step = ideal * (1 + info.eps / 2) + info.smallest_normal * info.eps
    assert bool(((groups - back).abs() <= step * (0.5 + 15 * info.eps / 2) * (1 + 2.0 ** -20)).all())
    assert bool((back[5, 0] == 0).all()) and bool((scales > 0).all())


@pytest.mark.parametrize('symmetric', [True, False])
@pytest.mark.parametrize('value', [float('nan'), float('inf'), -float('inf'), 1e6])
def test_weights_past_the_scales_are_refused(symmetric, value):
    w = torch.ones((4, 128))
    w[2, 70] = value
    with pytest.raises(ValueError, match='scale'):
        linear_w4.quantize_weight(w, 64, symmetric=symmetric)
    if value == 1e6:
        linear_w4.quantize_weight(w, 64, symmetric=symmetric, dtype=torch.bfloat16)
