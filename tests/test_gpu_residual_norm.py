"""residual_norm on the GPU: the update against its 64-bit statement, the norm
and codes bit for bit against norm_quantize of the updated rows."""
import pytest
import torch

from block_refs import assert_close, residual_update
from w8a8 import block_norm, convrot, kernels
from w8a8.h3_tensor_flow import StableNorm, labels_for, modulated_norm_quantize

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

CASES = [
    # rows, cols, x, branch, post norm, gate, modulation, codes (None, 'plain', 'rot', 'rot32', 'signs'), norm weight
    (1, 5120, F16, F16, False, False, False, None, True),
    (1, 16, BF16, F32, True, True, True, None, True),
    (3, 256, F16, F32, True, True, True, 'rot', True),
    (37, 1536, BF16, BF16, True, False, False, None, True),
    (130, 2064, F16, F16, True, True, False, None, True),      # 129 units: two and a bit lanes of units
    (65, 3584, F16, F16, False, True, True, 'rot', True),
    (29, 4096, BF16, F32, True, True, True, 'rot', True),
    (353, 5120, BF16, BF16, True, False, False, 'rot32', True),
    (201, 5376, F16, F32, False, True, True, 'rot', True),
    (1000, 5376, F16, F16, True, True, True, 'signs', True),
    (2050, 1024, F16, F16, True, True, True, 'plain', True),
    (2050, 5376, F16, F16, False, True, True, 'rot', True),
    (9, 6144, BF16, F32, True, True, True, 'plain', False),
    (5, 8192, F16, F16, True, True, True, 'rot', True),        # past six units a lane: the streaming passes
    (3, 8208, BF16, F32, True, False, True, None, False),
    (2, 16384, F16, F32, True, True, True, 'rot32', True),
    (4, 32, F16, F16, False, False, False, 'plain', False),
]


def _case(rows, cols, dt, bt, post, gate, mod, seed, gpu):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, cols), generator=g) * 0.05).to(dt)
    branch = (torch.randn((rows, cols), generator=g) * (3 if post else 0.05)).to(bt)
    if rows > 2:
        branch[1] = 0                                   # an all-zero branch: 1 / sqrt(eps)
        x[2], branch[2] = 0, 0                          # an all-zero row after the update
    kw = dict(branch_scale=1 / 512 if post else 1.0)
    if post:
        kw.update(post_eps=1e-6, post_weight=(torch.rand(cols, generator=g) + 0.5).to(gpu))
    table = {}
    if gate:
        kw['gate'] = torch.randn((5, cols), generator=g).to(gpu)
    if mod:
        table = dict(shift=(torch.randn((9, cols), generator=g) * 0.1).to(gpu),
                     scale=(torch.randn((9, cols), generator=g) * 0.1).to(gpu))
    labels = torch.randint(0, 9 if not gate else 5, (rows,), generator=g, dtype=torch.int32)
    if rows > 4:
        labels[3], labels[4] = -7, 1000                 # clamped into each table
    if gate or mod:
        kw['labels'] = labels.to(gpu)
    return x.to(gpu), branch.to(gpu), kw, table, (torch.rand(cols, generator=g) + 0.5).to(gpu)


def _bits(t):
    return t.view(torch.int16) if t.element_size() == 2 else t.view(torch.int8)


@pytest.mark.parametrize('rows,cols,dt,bt,post,gate,mod,codes,weight', CASES)
def test_update_and_norm(gpu, rows, cols, dt, bt, post, gate, mod, codes, weight):
    print(f'residual_norm {rows}x{cols} {dt} {bt} {post} {gate} {mod} {codes}', flush=True)
    x, branch, kw, table, w = _case(rows, cols, dt, bt, post, gate, mod, rows * 31 + cols, gpu)
    w = w if weight else None
    q = dict(quantize=codes is not None, convrot=codes not in (None, 'plain'), round_rotated=codes != 'rot32',
             signs=convrot.sign_words(convrot.signs(cols, 5), gpu) if codes == 'signs' else None)
    keep = x.clone(), branch.clone()
    r = block_norm.residual_norm(x, branch, weight=w, eps=1e-7, **kw, **table, want_normalized=True, **q)
    torch.cuda.synchronize()
    assert torch.equal(x, keep[0]) and torch.equal(branch, keep[1])
    exact, slack = residual_update(x, branch, **kw)
    assert_close(r['x'], exact, slack, 'updated rows')
    want = kernels.norm_quantize(r['x'], w, table.get('shift'), table.get('scale'), kw.get('labels') if table else None,
                                 eps=1e-7, want_normalized=True, **q)
    assert torch.equal(_bits(r['y']), _bits(want['y']))
    if codes is not None:
        assert torch.equal(r['q'], want['q'])
        assert torch.equal(r['scale'].view(torch.int32), want['scale'].view(torch.int32))
    # The update alone, the norm alone of the outputs and an update in place give the same rows.
    alone = block_norm.residual_norm(x, branch, **kw)
    assert set(alone) == {'x'} and torch.equal(_bits(alone['x']), _bits(r['x']))
    inplace = x.clone()
    again = block_norm.residual_norm(inplace, branch, weight=w, eps=1e-7, **kw, **table, out=inplace, **q)
    assert again['x'] is inplace and torch.equal(_bits(inplace), _bits(r['x']))
    for key in ('y', 'q', 'scale'):
        if key in again:
            assert torch.equal(again[key], r[key]), key


def test_rows_alone_equal_rows_of_a_batch(gpu):
    """The order of every sum is the row's own: no launch shape changes a bit."""
    rows, cols = 1800, 5376
    x, branch, kw, table, w = _case(rows, cols, F16, F32, True, True, True, 5, gpu)
    r = block_norm.residual_norm(x, branch, weight=w, eps=1e-7, **kw, **table, quantize=True, want_normalized=True)
    labels = kw.pop('labels')
    for lo, hi in ((0, 1), (3, 5), (700, 1030), (1799, 1800)):
        s = block_norm.residual_norm(x[lo:hi], branch[lo:hi], weight=w, eps=1e-7, labels=labels[lo:hi], **kw, **table,
                                     quantize=True, want_normalized=True)
        for key in r:
            assert torch.equal(s[key], r[key][lo:hi]), (key, lo, hi)


def test_matches_the_gated_epilogue(gpu):
    """Without a norm of the branch the update is the GEMM epilogue's: one FMA, one rounding."""
    g = torch.Generator().manual_seed(3)
    m, n, k = 77, 512, 256
    q = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8).to(gpu)
    wq = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).to(gpu)
    a, s = (torch.rand(m, generator=g) * 1e-2).to(gpu), (torch.rand(n, generator=g) * 1e-3).to(gpu)
    x = torch.randn((m, n), generator=g).half().to(gpu)
    gate = torch.randn((4, n), generator=g).to(gpu)
    labels = torch.randint(0, 4, (m,), generator=g, dtype=torch.int32).to(gpu)
    branch = kernels.gemm(q, wq, epilogue=kernels.EPI_ROW, row_scale=a, col_scale=s)
    for kw in (dict(gate=gate, labels=labels), {}):
        want = kernels.gemm(q, wq, epilogue=kernels.EPI_ROW, row_scale=a, col_scale=s, residual=x,
                            **(dict(gate=gate, gate_labels=labels) if kw else {}))
        got = block_norm.residual_norm(x, branch, **kw)['x']
        assert torch.equal(_bits(got), _bits(want))


def test_strided_rows_and_one_element_tables(gpu):
    g = torch.Generator().manual_seed(4)
    rows, cols = 70, 512
    big = torch.randn((rows, 3 * cols), generator=g).half().to(gpu)
    x, branch = big[:, :cols], big[:, cols:2 * cols]
    gate = torch.randn((2, 2 * cols), generator=g).to(gpu)[:, cols:]
    labels = (torch.arange(rows) % 2).int().to(gpu)
    r = block_norm.residual_norm(x, branch, eps=1e-6, gate=gate, labels=labels, out=big[:, 2 * cols:])
    want = block_norm.residual_norm(x.contiguous(), branch.contiguous(), eps=1e-6, gate=gate.contiguous(),
                                    labels=labels)
    assert torch.equal(r['x'], want['x']) and torch.equal(r['y'], want['y'])
    # Rows that do not start on 16 bytes, and a transposed branch, are copied.
    odd = torch.randn((rows, cols + 1), generator=g).half().to(gpu)[:, 1:]
    turned = torch.randn((cols, rows), generator=g).half().to(gpu).t()
    r = block_norm.residual_norm(odd, turned, eps=1e-6)
    want = block_norm.residual_norm(odd.clone(memory_format=torch.contiguous_format), turned.contiguous(), eps=1e-6)
    assert torch.equal(r['x'], want['x']) and torch.equal(r['y'], want['y'])
    empty = block_norm.residual_norm(x[:0], branch[:0], eps=1e-6, quantize=True)
    assert empty['x'].shape == (0, cols) and empty['q'].shape == (0, cols)


def test_special_values_stay_in_their_row(gpu):
    rows, cols = 12, 1024
    g = torch.Generator().manual_seed(6)
    x = torch.randn((rows, cols), generator=g).half()
    b = torch.randn((rows, cols), generator=g).half()
    clean = block_norm.residual_norm(x.to(gpu), b.to(gpu), eps=1e-6, post_eps=1e-6)
    b[2, 7], b[5, 0], x[8, 3] = float('nan'), float('inf'), float('-inf')
    r = block_norm.residual_norm(x.to(gpu), b.to(gpu), eps=1e-6, post_eps=1e-6)
    others = [i for i in range(rows) if i not in (2, 5, 8)]
    assert torch.equal(r['x'][others], clean['x'][others]) and torch.equal(r['y'][others], clean['y'][others])
    assert bool(torch.isnan(r['x'][2]).all())                       # a NaN branch element: its norm is NaN
    exact, _ = residual_update(x, b, post_eps=1e-6)
    for i in (5, 8):
        assert torch.equal(torch.isnan(r['x'][i].cpu()), torch.isnan(exact[i]))
        assert torch.equal(torch.isinf(r['x'][i].cpu()), torch.isinf(exact[i]))


def test_update_and_prepare(gpu):
    g = torch.Generator().manual_seed(7)
    rows, hidden = 200, 1024
    x = torch.randn((rows, hidden), generator=g).half().to(gpu)
    branch = torch.randn((rows, hidden), generator=g).to(gpu)
    gate, shift, scale = (torch.randn((9, hidden), generator=g).to(gpu) * 0.1 for _ in range(3))
    segments = [(0, 50, 2), (50, 199, 8), (199, 200, 0)]
    norm = StableNorm(torch.nn.RMSNorm(hidden, eps=1e-6, device=gpu), 512.0)
    post = torch.nn.RMSNorm(hidden, eps=1e-5, device=gpu)
    new, (q, s) = block_norm.update_and_prepare(x, branch, gate, segments, norm, shift, scale, post_norm=post,
                                                branch_scale=1 / 512)
    exact, slack = residual_update(x, branch, post_weight=post.weight.detach(), post_eps=1e-5, gate=gate,
                                   labels=labels_for(rows, segments, 9, device=gpu), branch_scale=1 / 512)
    assert_close(new, exact, slack, 'updated rows')
    wq, ws = modulated_norm_quantize(norm, new, shift, scale, segments)
    assert torch.equal(q, wq) and torch.equal(s, ws)


def test_refusals(gpu):
    x = torch.zeros((4, 256), dtype=F16, device=gpu)
    t = torch.zeros((2, 256), device=gpu)
    lab = torch.zeros(4, dtype=torch.int32, device=gpu)
    for a, kw in (((x.float(), x), {}), ((x, x.bfloat16()), {}), ((x, x[:2]), {}), ((x, x.cpu()), {}),
                  ((x, x), dict(quantize=True)), ((x, x), dict(weight=t[0])), ((x, x), dict(post_weight=t[0])),
                  ((x[:, :24], x[:, :24]), {}), ((x[:, :240], x[:, :240]), dict(eps=1e-6, quantize=True)),
                  ((x, x), dict(gate=t)), ((x, x), dict(gate=t, labels=lab.long())), ((x, x), dict(gate=t, labels=lab[:3])),
                  ((x, x), dict(gate=t[:, :128], labels=lab)), ((x, x), dict(gate=t.half(), labels=lab)),
                  ((x, x), dict(gate=t[:0], labels=lab)),
                  ((x, x), dict(eps=1e-6, shift=t)), ((x, x), dict(eps=1e-6, shift=t, scale=t[:1], labels=lab)),
                  ((x, x), dict(out=x[:2])), ((x, x), dict(out=x.float())), ((x, x), dict(eps=1e-6, weight=t)),
                  ((x, x), dict(eps=1e-6, signs=torch.zeros(256, dtype=torch.int32, device=gpu)))):
        with pytest.raises(ValueError):
            block_norm.residual_norm(*a, **kw)
    from w8a8._abi import W8A8Error
    with pytest.raises(W8A8Error, match='overlaps the branch'):
        block_norm.residual_norm(x.clone(), x, out=x)
