"""Calls of the operators around a block's projections without a GPU: refusals
and the 4-bit quantizer's range."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from w8a8 import _abi, axial_rope, block_norm, linear_w4


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


def _update_args(rows=4, hidden=256, table_rows=3):
    x = torch.zeros((rows, hidden), dtype=torch.float16)
    tables = [torch.zeros((table_rows, hidden)) for _ in range(3)]
    return [x, torch.zeros_like(x), tables[0], [(0, rows, 1)], torch.nn.RMSNorm(hidden, eps=1e-6), tables[1], tables[2]]


@pytest.mark.parametrize('which', [0, 1, 2, 5, 6])
def test_update_and_prepare_loses_no_gradient(which):
    args = _update_args()
    args[which] = args[which].requires_grad_()
    with pytest.raises(ValueError, match='no gradient'):
        block_norm.update_and_prepare(*args)
    with torch.no_grad(), pytest.raises(ValueError, match='HIP device'):
        block_norm.update_and_prepare(*args)


def test_outputs_that_want_a_gradient_are_refused():
    x = torch.zeros((2, 256), dtype=torch.float16)
    with pytest.raises(ValueError, match='no gradient'):
        block_norm.residual_norm(x, x.clone(), out=torch.zeros_like(x, requires_grad=True))
    out = torch.zeros((2, 16), dtype=torch.float16, requires_grad=True)
    with pytest.raises(ValueError, match='no gradient'):
        linear_w4.linear(x, torch.zeros((16, 32), dtype=torch.int32), torch.ones((2, 16), dtype=torch.float16), out=out)


def test_forward_mode_tangents_are_refused():
    """A dual tensor has requires_grad False, and no_grad does not stop its tangent."""
    x = torch.zeros((2, 256), dtype=torch.float16)
    q = torch.zeros((2, 4, 128), dtype=torch.float16)
    inv, axis = axial_rope.ladder((16, 16, 16))
    pos = torch.zeros((2, 3))
    codes, scales = torch.zeros((16, 32), dtype=torch.int32), torch.ones((2, 16), dtype=torch.float16)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: block_norm.residual_norm(dual(x), x, eps=1e-6),
                 lambda: block_norm.residual_norm(x, x, eps=1e-6, weight=dual(torch.ones(256))),
                 lambda: axial_rope.rotate(dual(q), None, pos, inv, axis),
                 lambda: axial_rope.rotate(q, None, dual(pos), inv, axis),
                 lambda: axial_rope.freqs(dual(pos), inv, axis),
                 lambda: linear_w4.linear(dual(x), codes, scales),
                 lambda: linear_w4.linear(x, codes, dual(scales))]
        for call in calls:
            with pytest.raises(ValueError, match='no gradient'):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match='no gradient'):
                call()
    with pytest.raises(ValueError, match='HIP device'):
        block_norm.residual_norm(x, x, eps=1e-6)


def test_modulation_tables_have_the_segments_rows():
    """The segments name one row of gate, shift and scale alike; a table may have others."""
    for which, change in ((2, lambda t: t[:1]), (5, lambda t: t[0]), (6, lambda t: None), (2, lambda t: None)):
        args = _update_args()
        args[which] = change(args[which])
        with pytest.raises(ValueError, match='table'):
            block_norm.update_and_prepare(*args)
    for rows in (2, 7):
        args = _update_args()
        args[2] = torch.zeros((rows, 256))
        with pytest.raises(ValueError, match='HIP device'):
            block_norm.update_and_prepare(*args)


@pytest.mark.parametrize('gated', [0, 1])
def test_few_rows_of_too_many_outputs_are_refused(gated):
    """Up to eight rows are one launch of n / 32 workgroups of 256 lanes: below 2^32."""
    args = _abi.LinearW4Args(dtype=_abi.F16, x=1 << 20, ldx=32, codes=1 << 41, ldw=4, scales=64, m=1, n=1 << 29, k=32,
                             group=32, gated=gated, out=1 << 40, ldo=1 << 29)
    args.struct_size = ctypes.sizeof(args)
    lib = _abi.load()
    assert lib.w8a8_linear_w4(ctypes.byref(args)) == _abi.ERR_INVALID
    assert 'too many outputs' in lib.w8a8_last_error().decode()


@pytest.mark.parametrize('first,second', [(0, 64), (0, 300), (128, 200)])
def test_interleaved_heads_that_overlap_are_refused(first, second):
    # q and k of [rows, heads, 3, dim]: k's channels may not run into q's.
    st = (3 * 4 * 128, 3 * 128)
    base = 1 << 20
    q, k = base + 2 * first, base + 2 * second
    args = _abi.AxialRopeArgs(dtype=_abi.F16, q=q, k=k, q_out=q, k_out=k, rows=5, q_heads=4, k_heads=4, dim=128,
                              pairs=64, axes=1, q_strides=st, k_strides=st, q_out_strides=st, k_out_strides=st,
                              positions=64, pos_strides=(1, 1), inv_freq=128, axis=256, eps=1e-6)
    args.struct_size = ctypes.sizeof(args)
    lib = _abi.load()
    assert lib.w8a8_axial_rope(ctypes.byref(args)) == _abi.ERR_INVALID
    assert 'overlap' in lib.w8a8_last_error().decode()
