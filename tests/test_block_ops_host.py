"""The operators around a block's projections without a GPU: argument checks of
the C entry points (nothing is launched), the ladder and grid builders, the
4-bit packing and its quantizer."""
import ctypes

import pytest
import torch

from w8a8 import _abi, axial_rope, block_norm, linear_w4


def _refused(name, args, fragment):
    lib = _abi.load()
    args.struct_size = ctypes.sizeof(args)
    assert getattr(lib, name)(ctypes.byref(args)) == _abi.ERR_INVALID
    assert fragment in lib.w8a8_last_error().decode(), lib.w8a8_last_error().decode()


def _accepted(name, args):
    lib = _abi.load()
    args.struct_size = ctypes.sizeof(args)
    assert getattr(lib, name)(ctypes.byref(args)) == _abi.OK, lib.w8a8_last_error().decode()


def test_struct_layouts():
    lib = _abi.load()
    assert [ctypes.sizeof(s) for s in _abi.BLOCK_STRUCTS] == [232, 208, 88, 152]
    for i, st in enumerate(_abi.BLOCK_STRUCTS):
        assert lib.w8a8_struct_size(8 + i) == ctypes.sizeof(st)
    for name, st in zip(_abi.BLOCK_ENTRY_POINTS, _abi.BLOCK_STRUCTS):
        a = st(struct_size=8)
        assert getattr(lib, name)(ctypes.byref(a)) == _abi.ERR_INVALID
        assert 'struct_size' in lib.w8a8_last_error().decode()
        assert getattr(lib, name)(None) == _abi.ERR_INVALID


NORM = dict(x_dtype=_abi.F16, x=1 << 20, ldx=256, rows=4, cols=256, branch=2 << 20, ldb=256, branch_dtype=_abi.F16,
            branch_scale=1.0, residual_scale=1.0, out=3 << 20, ldo=256, y=4 << 20, ldy=256, eps=1e-6)


@pytest.mark.parametrize('change,fragment', [
    (dict(x_dtype=_abi.F32), 'x_dtype'),
    (dict(branch_dtype=_abi.BF16), 'branch_dtype'),
    (dict(post=2), 'post'),
    (dict(post_weight=64), 'post_weight'),
    (dict(rows=-1), 'shape'),
    (dict(cols=24), 'multiple of 16'),
    (dict(cols=0), 'zero-width'),
    (dict(y=None, weight=64), 'without an output'),
    (dict(convrot=128), 'convrot'),
    (dict(round_rotated=2), 'round_rotated'),
    (dict(cols=240, ldx=240, convrot=256, q=5 << 20, q_scale=6 << 20, ldq=240), 'multiple of 256'),
    (dict(mod_shift=64), 'go together'),
    (dict(x=None), 'x must'),
    (dict(x=(1 << 20) + 8), 'x must'),
    (dict(ldx=252), 'x must'),
    (dict(ldx=260), 'x must'),
    (dict(branch=None), 'branch must'),
    (dict(branch_dtype=_abi.F32, ldb=258), 'branch must'),
    (dict(out=None), 'out must'),
    (dict(ldo=128), 'out must'),
    (dict(out=(1 << 20) + 64), 'overlaps x'),
    (dict(out=1 << 20, ldo=264), 'overlaps x'),
    (dict(out=2 << 20), 'overlaps the branch'),
    (dict(ldy=200), 'y must'),
    (dict(y=1 << 20), 'y overlaps'),
    (dict(y=3 << 20), 'y overlaps'),
    (dict(q=5 << 20, ldq=256), 'q_scale'),
    (dict(q=5 << 20, ldq=250, q_scale=6 << 20), 'q must'),
    (dict(q=1 << 20, ldq=256, q_scale=6 << 20), 'q or q_scale overlaps'),
    (dict(q=5 << 20, ldq=256, q_scale=3 << 20), 'q or q_scale overlaps'),
    (dict(weight=68), 'weights'),
    (dict(gate=64, gate_rows=2, ld_gate=256), 'labels'),
    (dict(gate=64, gate_rows=0, ld_gate=256, labels=64), 'gate must'),
    (dict(gate=64, gate_rows=2, ld_gate=254, labels=64), 'gate must'),
    (dict(mod_shift=64, mod_scale=128, mod_rows=1, ld_mod=256), 'labels'),
    (dict(mod_shift=64, mod_scale=128, mod_rows=0, ld_mod=256, labels=64), 'tables'),
    (dict(convrot_signs=64), 'convrot_signs'),
])
def test_residual_norm_refusals(change, fragment):
    _refused('w8a8_residual_norm', _abi.ResidualNormArgs(**{**NORM, **change}), fragment)


def test_empty_calls_do_nothing():
    _accepted('w8a8_residual_norm', _abi.ResidualNormArgs(**{**NORM, 'rows': 0, 'x': None, 'out': None}))
    _accepted('w8a8_axial_rope', _abi.AxialRopeArgs(**{**ROPE, 'rows': 0}))
    _accepted('w8a8_axial_freqs', _abi.AxialFreqsArgs(**{**FREQS, 'rows': 0}))
    _accepted('w8a8_linear_w4', _abi.LinearW4Args(**{**W4, 'm': 0, 'x': None}))
    _accepted('w8a8_linear_w4', _abi.LinearW4Args(**{**W4, 'n': 0, 'codes': None}))


ROPE = dict(dtype=_abi.F16, q=1 << 20, k=2 << 20, q_out=3 << 20, k_out=4 << 20, rows=4, q_heads=4, k_heads=2, dim=128,
            pairs=64, axes=3, q_strides=(512, 128), k_strides=(256, 128), q_out_strides=(512, 128),
            k_out_strides=(256, 128), positions=64, pos_strides=(3, 1), inv_freq=128, axis=256, eps=1e-6)


@pytest.mark.parametrize('change,fragment', [
    (dict(dtype=_abi.I8), 'dtype'),
    (dict(dim=127), 'dim'),
    (dict(dim=258), 'dim'),
    (dict(pairs=65), 'pairs'),
    (dict(pairs=0), 'pairs'),
    (dict(axes=0), 'axes'),
    (dict(axes=17), 'axes'),
    (dict(pairing=2), 'pairing'),
    (dict(pos_type=3), 'pos_type'),
    (dict(q_heads=0), 'heads'),
    (dict(k=None), 'go together'),
    (dict(k_heads=0), 'go together'),
    (dict(q_gain=64), 'q_gain and k_gain'),
    (dict(q=None), 'null'),
    (dict(positions=None), 'null'),
    (dict(positions=66), 'misaligned'),
    (dict(inv_freq=68), 'misaligned'),
    (dict(pos_strides=(-3, 1)), 'position stride'),
    (dict(q=(1 << 20) + 1), 'misaligned tensor'),
    (dict(q_strides=(-512, 128)), 'negative stride'),
    (dict(q_out_strides=(512, 64)), 'heads overlap'),
    (dict(q_out_strides=(256, 128)), 'heads overlap'),
    (dict(q_out=(1 << 20) + 128), 'overlaps an input'),
    (dict(q_out=2 << 20), 'overlaps an input'),
    (dict(q_out=1 << 20, q_out_strides=(520, 128)), 'overlaps an input'),
    (dict(k_out=3 << 20), 'q_out and k_out overlap'),
    (dict(rows=1 << 31), 'rows or heads'),
])
def test_axial_rope_refusals(change, fragment):
    _refused('w8a8_axial_rope', _abi.AxialRopeArgs(**{**ROPE, **change}), fragment)


def test_axial_rope_in_place_views_of_a_packed_row_that_overlap_are_refused():
    # q [4 heads] and k [2 heads] of one packed row of 8 heads: k may start at
    # head 4, not inside q's heads.
    row = dict(q_strides=(1024, 128), k_strides=(1024, 128), q_out_strides=(1024, 128), k_out_strides=(1024, 128))
    base = 1 << 20
    bad = {**ROPE, **row, 'q': base, 'q_out': base, 'k': base + 3 * 256, 'k_out': base + 3 * 256}
    _refused('w8a8_axial_rope', _abi.AxialRopeArgs(**bad), 'overlap')
    wraps = {**ROPE, **row, 'q': base, 'q_out': base, 'k': base + 7 * 256, 'k_out': base + 7 * 256}
    _refused('w8a8_axial_rope', _abi.AxialRopeArgs(**wraps), 'overlap')


FREQS = dict(freq_dtype=_abi.F16, positions=64, pos_strides=(3, 1), rows=4, pairs=48, axes=3, inv_freq=128, axis=256,
             freqs=4096)


@pytest.mark.parametrize('change,fragment', [
    (dict(freq_dtype=_abi.BF16), 'freq_dtype'), (dict(freq_layout=2), 'freq_layout'), (dict(pos_type=-1), 'pos_type'),
    (dict(pairs=0), 'range'), (dict(pairs=129), 'range'), (dict(axes=17), 'range'), (dict(rows=-1), 'range'),
    (dict(freqs=None), 'null'), (dict(freqs=4104), 'misaligned'), (dict(axis=258), 'misaligned'),
    (dict(pos_strides=(0, -1)), 'position stride'),
])
def test_axial_freqs_refusals(change, fragment):
    _refused('w8a8_axial_freqs', _abi.AxialFreqsArgs(**{**FREQS, **change}), fragment)


W4 = dict(dtype=_abi.F16, x=1 << 20, ldx=256, codes=2 << 20, ldw=32, scales=64, m=4, n=32, k=256, group=128,
          out=3 << 20, ldo=32)


@pytest.mark.parametrize('change,fragment', [
    (dict(dtype=_abi.F32), 'dtype'),
    (dict(gated=2), 'gated'),
    (dict(group=16), 'group'),
    (dict(group=0), 'group'),
    (dict(group=96), 'group'),
    (dict(group=192), 'group'),
    (dict(k=320, group=128, ldx=320, ldw=40), 'multiple of the group'),
    (dict(k=0), 'size'),
    (dict(m=-1), 'size'),
    (dict(m=1 << 22), 'size'),
    (dict(gated=1, n=33), 'gated'),
    (dict(gated=1, residual=64, ldr=32), 'gated'),
    (dict(x=None), 'x must'),
    (dict(x=(1 << 20) + 2), 'x must'),
    (dict(ldx=255), 'x must'),
    (dict(codes=(2 << 20) + 4), 'codes must'),
    (dict(ldw=30), 'codes must'),
    (dict(scales=None), 'scales'),
    (dict(residual=64, ldr=31), 'residual'),
    (dict(out=None), 'out'),
    (dict(ldo=31), 'out'),
    (dict(out=1 << 20), 'overlaps x'),
    (dict(residual=(3 << 20) + 2, ldr=32), 'overlaps the residual'),
])
def test_linear_w4_refusals(change, fragment):
    _refused('w8a8_linear_w4', _abi.LinearW4Args(**{**W4, **change}), fragment)


@pytest.mark.parametrize('change', [dict(ldw=1 << 22), dict(ldx=1 << 22), dict(n=1 << 30, ldo=1 << 30)])
def test_linear_w4_many_rows_offsets_fit_32_bits(change):
    case = {**W4, **change, 'm': 16, 'x': 1 << 50, 'out': 1 << 40, 'workspace': 1 << 45, 'workspace_bytes': 1 << 40}
    _refused('w8a8_linear_w4', _abi.LinearW4Args(**case), 'too long')


@pytest.mark.parametrize('group', [0, -128, 16, 192])
def test_group_sizes_are_refused(group):
    with pytest.raises(ValueError):
        linear_w4.quantize_weight(torch.zeros((4, 768)), group)
    with pytest.raises(ValueError):
        linear_w4.LinearW4(768, 4, group_size=group, device='cpu')


@pytest.mark.parametrize('features,kw', [(0, {}), (100, {}), (256, dict(dtype=torch.float32)),
                                         (256, dict(gated=True))])
def test_modules_are_refused(features, kw):
    with pytest.raises(ValueError):
        linear_w4.LinearW4(features, 5, device='cpu', **kw)


def test_cpu_tensors_are_refused():
    x = torch.zeros((2, 256), dtype=torch.float16)
    with pytest.raises(ValueError):
        block_norm.residual_norm(x, x, eps=1e-6)
    inv, axis = axial_rope.ladder((16, 16, 16))
    pos = torch.zeros((2, 3), dtype=torch.int64)
    q = torch.zeros((2, 4, 128), dtype=torch.float16)
    with pytest.raises(ValueError):
        axial_rope.rotate(q, q, pos, inv, axis)
    with pytest.raises(ValueError):
        axial_rope.rotate(q, q, pos, inv, axis, pairing='other')
    with pytest.raises(ValueError):
        axial_rope.freqs(pos, inv, axis)
    codes, scales, _ = linear_w4.quantize_weight(torch.randn((16, 256)))
    with pytest.raises(ValueError):
        linear_w4.linear(x, codes, scales)


def test_inputs_that_want_a_gradient_are_refused():
    x = torch.zeros((2, 256), dtype=torch.float16, requires_grad=True)
    with pytest.raises(ValueError, match='no gradient'):
        block_norm.residual_norm(x, x, eps=1e-6)
    with pytest.raises(ValueError, match='no gradient'):
        linear_w4.linear(x, torch.zeros((16, 32), dtype=torch.int32), torch.ones((2, 16), dtype=torch.float16))
    q = torch.zeros((2, 4, 128), dtype=torch.float16, requires_grad=True)
    inv, axis = axial_rope.ladder((16, 16, 16))
    with pytest.raises(ValueError, match='no gradient'):
        axial_rope.rotate(q, None, torch.zeros((2, 3), dtype=torch.int64), inv, axis)


def test_ladders():
    inv, axis = axial_rope.ladder((2, 3, 1), theta=100.0)
    assert axis.tolist() == [0, 0, 1, 1, 1, 2] and inv.dtype == torch.float64
    assert inv.tolist() == pytest.approx([1, 0.1, 1, 100 ** (-1 / 3), 100 ** (-2 / 3), 1])
    inv, axis = axial_rope.ladder((2, 3, 1), theta=100.0, shared=True)
    assert axis.tolist() == [0, 0, 1, 1, 1, 2]
    assert inv.tolist() == pytest.approx([100 ** (-p / 6) for p in range(6)])
    _, axis = axial_rope.ladder((24, 20, 20), shared=True, interleaved=True)
    assert axis.tolist() == [0, 1, 2] * 20 + [0] * 4
    _, axis = axial_rope.ladder((4,), shared=True, interleaved=True)
    assert axis.tolist() == [0] * 4
    for bad in (dict(sections=()), dict(sections=(0, 0)), dict(sections=(129,)), dict(sections=(-1, 3)),
                dict(sections=(8, 8), interleaved=True), dict(sections=(1, 7), shared=True, interleaved=True)):
        with pytest.raises(ValueError):
            axial_rope.ladder(**bad)


def test_grid_positions():
    p = axial_rope.grid_positions(2, 3, 4, start=(5, 0, 1))
    assert p.shape == (24, 3) and p.dtype == torch.int32
    assert p[0].tolist() == [5, 0, 1] and p[1].tolist() == [5, 0, 2] and p[4].tolist() == [5, 1, 1]
    assert p[-1].tolist() == [6, 2, 4]


def test_pack_layout_and_round_trip():
    c = torch.arange(16).repeat(3, 2)
    w = linear_w4.pack(c)
    assert w.shape == (3, 4) and w.dtype == torch.int32
    word = int(w[0, 0]) & 0xffffffff
    assert [(word >> (4 * i)) & 15 for i in range(8)] == [0, 2, 4, 6, 1, 3, 5, 7]
    assert torch.equal(linear_w4.unpack(w), c.to(torch.uint8))
    g = torch.Generator().manual_seed(1)
    c = torch.randint(0, 16, (5, 64), generator=g)
    assert torch.equal(linear_w4.unpack(linear_w4.pack(c)), c.to(torch.uint8))
    for bad in (c[:, :63], c + 9, c - 1, c.float()):
        with pytest.raises(ValueError):
            linear_w4.pack(bad)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('symmetric', [True, False])
def test_quantize_weight_is_within_half_a_step(dtype, symmetric):
    g = torch.Generator().manual_seed(2)
    w = torch.randn((24, 256), generator=g) * 0.05
    w[3, :64] = 0                                   # an all-zero group
    w[4, :64] = w[4, :64].abs()                     # one sign only
    codes, scales, zeros = linear_w4.quantize_weight(w, 64, symmetric=symmetric, dtype=dtype)
    assert codes.shape == (24, 32) and scales.shape == (4, 24) and scales.dtype == dtype
    assert (zeros is None) == symmetric
    back = linear_w4.dequantize_weight(codes, scales, zeros)
    step = scales.float().t().repeat_interleave(64, 1)
    # Half a step inside the code range; rounding the scale to its type moves
    # the range's ends (15 steps at most) by 15 half steps of that type.
    assert bool(((w - back).abs() <= step * (0.5 + 15 * torch.finfo(dtype).eps)).all())
    assert bool((back[3, :64] == 0).all())
    for bad in (dict(group_size=48), dict(group_size=512), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            linear_w4.quantize_weight(w, **bad)
