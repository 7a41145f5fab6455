"""Rotary positions with several axes on the GPU against their 64-bit statement."""
import pytest
import torch

from block_refs import assert_close, half_step, rope
from w8a8 import axial_rope, kernels, rms_rope

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

CASES = [
    # rows, heads, k heads, dim, sections, options of the ladder, dtype, norm, adjacent, position type, farthest
    (1, 64, 8, 128, (24, 20, 20), dict(shared=True, interleaved=True), F16, True, False, torch.int64, 262144),
    (1, 1, 0, 2, (1,), {}, F32, False, False, torch.int32, 10),
    (353, 16, 2, 128, (24, 20, 20), dict(shared=True, interleaved=True), BF16, True, False, torch.int64, 1000),
    (37, 28, 28, 128, (16, 16, 16), {}, F16, True, False, torch.int32, 80),          # a prefix of 96 channels
    (70, 3, 1, 72, (18, 18), {}, F32, False, False, torch.int64, 64),                # chunks of 4, lanes to spare
    (70, 3, 1, 72, (18, 18), {}, F16, True, True, torch.float32, 64),
    (19, 5, 5, 80, (10, 10, 10, 10), dict(shared=True), BF16, True, True, torch.int32, 5000),
    (11, 2, 2, 256, (128,), {}, F32, True, False, torch.int64, 1000000),             # 128 pairs of one axis
    (11, 2, 2, 256, (37,), {}, F16, True, False, torch.int64, 1000000),              # odd pairs: chunks of one
    (11, 3, 3, 254, (60, 67), {}, BF16, True, True, torch.int64, 100),
    (9, 4, 2, 66, (5, 7, 21), {}, F16, False, False, torch.int32, 300),
    (2049, 4, 4, 64, (8, 12, 12), {}, BF16, False, True, torch.float32, 200),
    (600, 28, 28, 128, (16, 16, 16), {}, F16, True, True, torch.int32, 80),
    (33, 7, 1, 96, (6, 6), {}, F32, True, False, torch.int64, 20000),
    (5, 2, 1, 128, (4,) * 16, {}, F16, False, False, torch.int32, 50),               # sixteen axes
]


def _inputs(rows, heads, kheads, dim, sections, options, dtype, norm, ptype, far, gpu):
    g = torch.Generator().manual_seed(rows * 7 + dim + heads)
    q = (torch.randn((rows, heads, dim), generator=g) * 2).to(dtype)
    k = (torch.randn((rows, kheads, dim), generator=g) * 2).to(dtype) if kheads else None
    q[0, 0] = 0                                        # an all-zero head
    pos = torch.randint(0, far + 1, (rows, len(sections)), generator=g)
    pos[0, 0] = far
    pos = pos.to(ptype)
    if ptype == torch.float32:
        pos = pos / 4                                  # positions between the integers
    inv, axis = axial_rope.ladder(sections, **options)
    gains = [torch.rand(dim, generator=g) + 0.5 if norm else None for _ in range(2)]
    if k is None:
        gains[1] = None
    return [t.to(gpu) if t is not None else None for t in (q, k, pos, inv, axis, *gains)]


@pytest.mark.parametrize('rows,heads,kheads,dim,sections,options,dtype,norm,adjacent,ptype,far', CASES)
def test_rotate(gpu, rows, heads, kheads, dim, sections, options, dtype, norm, adjacent, ptype, far):
    print(f'rotate {rows}x{heads}+{kheads}x{dim} {sections} {dtype} norm={norm} adjacent={adjacent}', flush=True)
    q, k, pos, inv, axis, gq, gk = _inputs(rows, heads, kheads, dim, sections, options, dtype, norm, ptype, far, gpu)
    keep = q.clone()
    pairing = 'adjacent' if adjacent else 'half'
    kw = dict(pairing=pairing, q_gain=gq, k_gain=gk, eps=1e-5)
    qo, ko = axial_rope.rotate(q, k, pos, inv, axis, **kw)
    torch.cuda.synchronize()
    assert torch.equal(q, keep)
    for got, x, gain in ((qo, q, gq), (ko, k, gk)):
        if x is None:
            assert got is None
            continue
        exact, slack = rope(x, pos, inv, axis, adjacent=adjacent, gain=gain, eps=1e-5)
        assert_close(got, exact, slack, pairing)
    # In place, and with the heads of a [heads, rows, dim] buffer, the same bits.
    q2, k2 = q.clone(), k.clone() if k is not None else None
    axial_rope.rotate(q2, k2, pos, inv, axis, **kw, out=(q2, k2))
    assert torch.equal(q2, qo) and (k is None or torch.equal(k2, ko))
    turned = torch.full((heads, rows, dim), float('nan'), dtype=dtype, device=gpu)
    view = q.transpose(0, 1).contiguous().transpose(0, 1)
    axial_rope.rotate(view, None, pos, inv, axis, pairing=pairing, q_gain=gq, eps=1e-5, out=(turned.transpose(0, 1), None))
    assert torch.equal(turned.transpose(0, 1), qo)


def test_packed_rows_in_place_leave_v_alone(gpu):
    g = torch.Generator().manual_seed(1)
    rows, heads, kheads, dim = 130, 8, 2, 128
    packed = torch.randn((rows, (heads + 2 * kheads) * dim + 24), generator=g).half().to(gpu)
    before = packed.clone()

    def views(t):
        q, k = t[:, :heads * dim], t[:, heads * dim:(heads + kheads) * dim]
        return q.unflatten(1, (heads, dim)), k.unflatten(1, (kheads, dim))
    pos = torch.randint(0, 500, (3, rows), generator=g).to(gpu).t()           # [3, rows], as a strided view
    inv, axis = axial_rope.ladder((24, 20, 20), shared=True, interleaved=True, device=gpu)
    q, k = views(packed)
    want = axial_rope.rotate(q.contiguous(), k.contiguous(), pos.contiguous(), inv, axis)
    axial_rope.rotate(q, k, pos, inv, axis, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(packed[:, (heads + kheads) * dim:], before[:, (heads + kheads) * dim:])
    # Rows at an odd address: narrower loads, the same values.
    odd = torch.empty(rows * heads * dim + 1, dtype=torch.float16, device=gpu)[1:].view(rows, heads, dim)
    odd.copy_(views(before)[0])
    assert torch.equal(axial_rope.rotate(odd, None, pos, inv, axis)[0], want[0])


@pytest.mark.parametrize('dtype', [F16, F32])
@pytest.mark.parametrize('sections,rows', [((16, 16, 16), 1001), ((5,), 3), ((64, 64), 70)])
def test_freqs(gpu, dtype, sections, rows):
    g = torch.Generator().manual_seed(rows)
    pos = torch.randint(0, 100000, (rows, len(sections)), generator=g).to(gpu)
    inv, axis = axial_rope.ladder(sections, device=gpu)
    f = axial_rope.freqs(pos, inv, axis, dtype=dtype)
    n = sum(sections)
    assert f.shape == (1, rows, 1, n, 2, 2)
    phi = pos.double()[:, axis.long()] * inv
    exact = torch.stack([phi.cos(), -phi.sin(), phi.sin(), phi.cos()], -1).reshape(1, rows, 1, n, 2, 2)
    # The fraction of a turn in fp32 (half a turn: 2^-26 of one, times 2 pi) and
    # the series (2^-24): under 2^-22.
    assert_close(f, exact, torch.full_like(exact, 2.0 ** -22), 'freqs')
    assert torch.equal(axial_rope.freqs_pairs(pos, inv, axis, dtype=dtype), rms_rope.pack_freqs(f))


def test_freqs_feed_the_rms_rope(gpu):
    """The table through rms_rope and the positions through rotate agree to the
    table's rounding."""
    g = torch.Generator().manual_seed(2)
    rows, heads = 90, 4
    packed = torch.randn((rows, 3 * heads * 128), generator=g).half().to(gpu)
    pos = axial_rope.grid_positions(3, 5, 6, device=gpu)
    inv, axis = axial_rope.ladder((16, 16, 16), device=gpu)
    gq, gk = (torch.rand(128, generator=g).to(gpu) + 0.5 for _ in range(2))
    want = rms_rope.execute(packed, axial_rope.freqs(pos, inv, axis, dtype=F32), gq, gk, heads=heads, out_dtype=F16)
    q, k = (t.unflatten(1, (heads, 128)) for t in packed.split(heads * 128, 1)[:2])
    got = axial_rope.rotate(q, k, pos, inv, axis, q_gain=gq, k_gain=gk)
    for a, b in zip(got, want):
        size = b.double().abs() + 1e-3
        # Each is within half an fp16 step (and fp32 errors) of the exact value.
        assert bool(((a.double() - b.double()).abs() <= 2.1 * half_step(F16) * size + 2.0 ** -18).all())


def test_far_and_special_positions(gpu):
    """Angles of millions of radians keep their fraction; a position that is
    not finite makes its own pairs NaN and no others."""
    rows = 6
    pos = torch.tensor([[0.0], [16777216.0], [-3000000.0], [float('inf')], [float('nan')], [1e30]], device=gpu)
    inv, axis = axial_rope.ladder((32,), device=gpu)
    g = torch.Generator().manual_seed(5)
    q = torch.randn((rows, 2, 64), generator=g).to(gpu)
    got, _ = axial_rope.rotate(q, None, pos, inv, axis)
    exact, slack = rope(q[:3], pos[:3], inv, axis)
    assert_close(got[:3], exact, slack)
    assert torch.equal(got[0], q[0])
    assert bool(torch.isnan(got[3:5]).all())
    assert bool(torch.isfinite(got[5]).all())            # fp64 has no fraction left there, but a bounded turn
    assert bool((got[5].abs() <= 1.001 * (q[5, :, :32].abs() + q[5, :, 32:].abs()).repeat(1, 2)).all())


def test_launch_shape_changes_no_bit(gpu):
    g = torch.Generator().manual_seed(9)
    q = torch.randn((3000, 6, 128), generator=g).half().to(gpu)
    pos = torch.randint(0, 5000, (3000, 3), generator=g).to(gpu)
    inv, axis = axial_rope.ladder((16, 16, 16), device=gpu)
    gain = (torch.rand(128, generator=g) + 0.5).to(gpu)
    whole, _ = axial_rope.rotate(q, None, pos, inv, axis, q_gain=gain)
    for lo, hi in ((0, 1), (7, 20), (1000, 1700)):
        part, _ = axial_rope.rotate(q[lo:hi], None, pos[lo:hi], inv, axis, q_gain=gain)
        assert torch.equal(part, whole[lo:hi])


def test_refusals(gpu):
    q = torch.zeros((4, 2, 64), dtype=F16, device=gpu)
    pos = torch.zeros((4, 2), dtype=torch.int64, device=gpu)
    inv, axis = axial_rope.ladder((16, 16), device=gpu)
    gain = torch.ones(64, device=gpu)
    ok = dict(q=q, k=q.clone(), positions=pos, inv_freq=inv, axis=axis)
    for change in (dict(q=q.double()), dict(k=q.float()), dict(q=q[0]), dict(k=q[:3]), dict(k=q[..., :32]),
                   dict(q=q[:, :0]), dict(q=q[..., :63], k=None), dict(positions=pos[:3]), dict(positions=pos.half()),
                   dict(positions=pos[:, :0]), dict(positions=pos[0]), dict(inv_freq=inv[:5]), dict(inv_freq=inv.half()),
                   dict(axis=axis.long()), dict(q=q[..., :32], k=None), dict(q_gain=gain), dict(k_gain=gain),
                   dict(q_gain=gain[:32], k_gain=gain), dict(q_gain=gain.half(), k_gain=gain), dict(positions=pos.cpu()),
                   dict(out=(q, None)), dict(out=(q[:2], q[:2])), dict(out=(q.float(), q.float()))):
        with pytest.raises(ValueError):
            axial_rope.rotate(**{**ok, **change})
    from w8a8._abi import W8A8Error
    for change in (dict(out=(q, q)), dict(k=q, out=(q.clone(), q))):
        with pytest.raises(W8A8Error, match='overlap'):
            axial_rope.rotate(**{**ok, **change})
