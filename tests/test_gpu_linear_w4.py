"""4-bit projections on the GPU against their 64-bit statement."""
import pytest
import torch

from block_refs import assert_close, half_step, linear_w4 as exact_w4
from w8a8 import linear_w4

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16

CASES = [
    # m, n, k, group, dtype, zeros, bias, residual, gated
    (1, 1, 32, 32, F16, False, False, False, False),
    (1, 4096, 4096, 128, F16, False, False, False, False),
    (1, 2 * 1000, 1024, 128, BF16, True, True, False, True),
    (2, 33, 96, 32, BF16, True, True, True, False),
    (3, 130, 320, 64, F16, True, False, True, False),
    (5, 2, 256, 256, F16, False, True, False, True),
    (16, 512, 1152, 128, BF16, False, False, True, False),
    (17, 500, 2560, 128, F16, True, True, False, True),
    (31, 77, 512, 512, BF16, True, False, False, False),
    (33, 1030, 384, 64, F16, False, True, True, False),
    (64, 1024, 3584, 128, BF16, True, False, True, False),
    (65, 300, 640, 32, F16, True, True, False, False),
    (100, 2 * 129, 256, 128, BF16, False, False, False, True),
    (127, 257, 1024, 64, BF16, False, True, True, False),
    (128, 512, 512, 128, F16, True, False, False, False),
    (200, 2 * 300, 768, 256, F16, False, True, False, True),
    (353, 640, 1280, 128, F16, True, False, True, False),
    (353, 2 * 320, 1280, 64, BF16, True, True, False, True),
    (300, 1000, 96, 32, F16, False, False, False, False),
    (1025, 264, 384, 128, BF16, False, True, False, False),
]


def _case(m, n, k, group, dtype, zeros, bias, residual, gpu, seed=0):
    g = torch.Generator().manual_seed(seed + m * 131 + n * 7 + k)
    x = torch.randn((m, k), generator=g)
    x[:, 3] *= 20
    codes = torch.randint(0, 16, (n, k), generator=g)
    codes[0] = 15
    if n > 1:
        codes[1] = 0
    groups = k // group
    s = dict(x=x.to(dtype), scales=((torch.rand((groups, n), generator=g) + 0.1) * 0.02).to(dtype),
             zeros=torch.randint(0, 16, (groups, n), generator=g).to(torch.uint8) if zeros else None,
             bias=torch.randn(n, generator=g).to(dtype) if bias else None,
             residual=torch.randn((m, n), generator=g).to(dtype) if residual else None)
    return codes.to(gpu), {key: t.to(gpu) if t is not None else None for key, t in s.items()}


def _call(codes, s, gated=False, **kw):
    return linear_w4.linear(s['x'], linear_w4.pack(codes), s['scales'], s['zeros'], bias=s['bias'],
                            residual=s['residual'], gated=gated, **kw)


@pytest.mark.parametrize('m,n,k,group,dtype,zeros,bias,residual,gated', CASES)
def test_linear_w4(gpu, m, n, k, group, dtype, zeros, bias, residual, gated):
    print(f'linear_w4 {m}x{n}x{k} group {group} {dtype} {zeros} {bias} {residual} {gated}', flush=True)
    codes, s = _case(m, n, k, group, dtype, zeros, bias, residual, gpu)
    y = _call(codes, s, gated)
    torch.cuda.synchronize()
    exact, slack = exact_w4(s['x'], codes, s['scales'], s['zeros'], bias=s['bias'], residual=s['residual'], gated=gated)
    assert_close(y, exact, slack, 'outputs')
    off = float((y.double() - exact).norm() / exact.norm())
    assert off <= half_step(dtype) + 2.0 ** -16, off      # the rounding is nearly all of the error
    # Into a strided output whose margins stay as they were; a call gives the same bits again.
    width = n // 2 if gated else n
    wide = torch.full((m + 1, width + 7), 3.0, dtype=dtype, device=gpu)
    _call(codes, s, gated, out=wide[:m, 3:3 + width])
    assert torch.equal(wide[:m, 3:3 + width], y)
    wide[:m, 3:3 + width] = 3.0
    assert bool((wide == 3.0).all())


@pytest.mark.parametrize('group,dtype,k', [(128, F16, 1408), (128, BF16, 1536), (64, BF16, 1472), (64, F16, 2048),
                                           (32, BF16, 1376), (32, F16, 1056)])
@pytest.mark.parametrize('m', [8, 9, 32, 33, 64, 65, 129])
def test_where_the_kernels_change(gpu, m, group, dtype, k):
    # Odd and even numbers of 128-input steps, whole or not, split over k (few outputs).
    print(f'linear_w4 {m} rows, k {k} group {group} {dtype}', flush=True)
    codes, s = _case(m, 200, k, group, dtype, True, True, True, gpu)
    y = _call(codes, s)
    exact, slack = exact_w4(s['x'], codes, s['scales'], s['zeros'], bias=s['bias'], residual=s['residual'])
    assert_close(y, exact, slack, 'outputs')


@pytest.mark.parametrize('n,dtype,residual,gated', [(35837, F16, True, False), (35830, BF16, False, True)])
def test_more_tiles_than_a_round(gpu, n, dtype, residual, gated):
    # Whole tiles first, the last round's in ranges of k: 2 x 140 tiles of 128 x 256.
    print(f'linear_w4 130x{n}x1024 {dtype} {residual} {gated}', flush=True)
    codes, s = _case(130, n, 1024, 128, dtype, True, True, residual, gpu)
    y = _call(codes, s, gated)
    exact, slack = exact_w4(s['x'], codes, s['scales'], s['zeros'], bias=s['bias'], residual=s['residual'], gated=gated)
    assert_close(y, exact, slack, 'outputs')
    assert torch.equal(y, _call(codes, s, gated))


def test_broadcast_residual(gpu):
    codes, s = _case(5, 64, 256, 128, F16, False, False, True, gpu)
    row = s['residual'][:1]
    y = _call(codes, {**s, 'residual': row.expand(5, 64)})
    assert torch.equal(y, _call(codes, {**s, 'residual': row.repeat(5, 1)}))


def test_rows_of_ones_and_single_inputs(gpu):
    """Each weight alone: x a unit vector picks out one column of the weight, exactly."""
    g = torch.Generator().manual_seed(1)
    n, k, group = 48, 256, 64
    codes = torch.randint(0, 16, (n, k), generator=g)
    scales = (2.0 ** -torch.randint(0, 6, (k // group, n), generator=g).float()).half()
    zeros = torch.randint(0, 16, (k // group, n), generator=g).to(torch.uint8)
    w = (codes.reshape(n, -1, group) - zeros.t()[:, :, None]).float() * scales.float().t()[:, :, None]
    for dtype in (F16, BF16):
        eye = torch.eye(k, dtype=dtype, device=gpu)
        y = linear_w4.linear(eye, linear_w4.pack(codes).to(gpu), scales.to(dtype).to(gpu), zeros.to(gpu))
        assert torch.equal(y.float().cpu(), w.reshape(n, k).t())
        for row in (0, 100, 255):
            one = linear_w4.linear(eye[row:row + 1], linear_w4.pack(codes).to(gpu), scales.to(dtype).to(gpu), zeros.to(gpu))
            assert torch.equal(one.float().cpu(), w.reshape(n, k)[:, row][None])


def test_views_shapes_and_in_place_residual(gpu):
    codes, s = _case(12, 72, 256, 128, F16, True, True, True, gpu)
    want = _call(codes, s)
    words = linear_w4.pack(codes)
    lead = linear_w4.linear(s['x'].view(3, 4, 256), words, s['scales'], s['zeros'], bias=s['bias'],
                            residual=s['residual'].view(3, 4, 72))
    assert lead.shape == (3, 4, 72) and torch.equal(lead.view(12, 72), want)
    vector = linear_w4.linear(s['x'][5], words, s['scales'], s['zeros'], bias=s['bias'], residual=s['residual'][5])
    assert vector.shape == (72,)
    big = torch.zeros((12, 300), dtype=F16, device=gpu)
    big[:, 8:264] = s['x']
    assert torch.equal(_call(codes, {**s, 'x': big[:, 8:264]}), want)
    big[:, 7:263] = s['x']                               # rows off 16 bytes are copied
    assert torch.equal(_call(codes, {**s, 'x': big[:, 7:263]}), want)
    res = s['residual'].clone()
    assert linear_w4.linear(s['x'], words, s['scales'], s['zeros'], bias=s['bias'], residual=res, out=res) is res
    assert torch.equal(res, want)
    assert linear_w4.linear(s['x'][:0], words, s['scales'], s['zeros']).shape == (0, 72)


def test_rows_do_not_touch_each_other(gpu):
    """NaN and infinity in one row of x (padding of a batch) stay in it."""
    for m in (5, 40, 200):
        codes, s = _case(m, 96, 256, 128, BF16, False, False, False, gpu)
        want = _call(codes, s)
        s['x'][2] = float('nan')
        s['x'][m - 1] = float('inf')
        got = _call(codes, s)
        rows = [i for i in range(m) if i not in (2, m - 1)]
        assert torch.equal(got[rows], want[rows])
        assert bool(torch.isnan(got[2]).all()) and not bool(torch.isfinite(got[m - 1]).any())


def test_module(gpu):
    g = torch.Generator().manual_seed(3)
    w, b = torch.randn((512, 256), generator=g) * 0.05, torch.randn(512, generator=g)
    x = torch.randn((7, 256), generator=g).half().to(gpu)
    for kw in (dict(), dict(zeros=True, group_size=64), dict(bias=True), dict(gated=True, group_size=32, zeros=True)):
        mod = linear_w4.LinearW4(256, 512, device=gpu, **kw).load_weight(w.to(gpu), b.to(gpu) if 'bias' in kw else None)
        y = mod(x)
        back = linear_w4.dequantize_weight(mod.codes, mod.scales, mod.zeros).double()
        exact = x.double() @ back.t() + (mod.bias.double() if mod.bias is not None else 0)
        if mod.gated:
            a, u = exact.chunk(2, -1)
            exact = a * torch.sigmoid(a) * u
        assert float((y.double() - exact).norm() / exact.norm()) < half_step(F16) + 2.0 ** -16
        assert float((back - w.to(gpu).double()).norm() / w.double().norm()) < 0.15      # 4 bits of it


def test_refusals(gpu):
    codes, s = _case(4, 64, 256, 128, F16, True, True, True, gpu)
    words = linear_w4.pack(codes)
    ok = dict(x=s['x'], codes=words, scales=s['scales'], zeros=s['zeros'], bias=s['bias'], residual=s['residual'])
    for change in (dict(x=s['x'].float()), dict(x=s['x'][:, :128]), dict(codes=codes), dict(codes=words.long()),
                   dict(scales=s['scales'].float()), dict(scales=s['scales'].bfloat16()), dict(scales=s['scales'][:, :32]),
                   dict(scales=torch.zeros((3, 64), dtype=F16, device=gpu)),
                   dict(scales=torch.zeros((16, 64), dtype=F16, device=gpu), zeros=None),
                   dict(zeros=s['zeros'].int()), dict(zeros=s['zeros'][:1]), dict(bias=s['bias'].float()),
                   dict(bias=s['bias'][:3]), dict(residual=s['residual'].float()), dict(residual=s['residual'][:2]),
                   dict(gated=True), dict(out=torch.zeros((4, 63), dtype=F16, device=gpu)),
                   dict(out=torch.zeros((4, 64), device=gpu)), dict(codes=words.cpu())):
        with pytest.raises(ValueError):
            linear_w4.linear(**{**ok, **change})
    from w8a8._abi import W8A8Error
    big = torch.zeros((4, 256), dtype=F16, device=gpu)
    with pytest.raises(W8A8Error, match='overlaps x'):
        linear_w4.linear(big, words, s['scales'], out=big[:, :64])
