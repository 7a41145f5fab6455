"""Every kernel that the operators around a block's projections choose by size,
type or mode, by the checks of each operator's own tests."""
import pytest
import torch

import test_gpu_linear_w4 as w4
import test_gpu_residual_norm as norm
from block_refs import assert_close, linear_w4 as exact_w4
from w8a8 import block_norm, kernels

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize('rows,cols,dt,bt,post,gate,mod,codes,weight', [
    # More than 768 rows, whose labels differ from row to row within a workgroup: 1 to
    # 6 units a lane, whole and ragged, each mode, both types and both branches.
    (769, 1008, F16, F16, True, True, True, None, True),
    (900, 1024, BF16, F32, True, False, True, 'rot32', True),
    (1031, 2048, F16, F32, False, True, False, 'plain', True),
    (800, 2064, BF16, BF16, True, True, True, None, True),
    (801, 2816, F16, F16, True, True, True, 'rot', True),
    (770, 2832, BF16, F32, True, True, True, None, False),
    (1300, 3584, BF16, BF16, False, True, True, 'rot', True),
    (777, 4096, F16, F16, True, True, True, 'rot32', True),
    (850, 4864, BF16, BF16, True, True, True, 'plain', True),
    (1025, 5120, BF16, BF16, True, False, False, None, True),
    (1025, 5120, F16, F32, True, True, True, 'rot32', True),
    (1537, 5376, F16, F16, True, True, True, None, True),
    (769, 5376, BF16, BF16, True, True, True, 'rot32', True),
    (1100, 5376, BF16, F32, True, True, True, 'rot', True),
    (900, 6144, F16, F16, True, True, True, 'signs', True),     # the most that is staged
    (900, 6144, BF16, F32, True, True, True, None, True),
    # At 768 rows a workgroup has a row.
    (768, 5376, BF16, F32, True, True, True, 'rot32', True),
    (768, 2832, F16, F16, True, True, True, None, True),
])
def test_residual_norm_rows(gpu, rows, cols, dt, bt, post, gate, mod, codes, weight):
    norm.test_update_and_norm(gpu, rows, cols, dt, bt, post, gate, mod, codes, weight)


@pytest.mark.parametrize('dt', [F16, BF16])
@pytest.mark.parametrize('codes', [False, True])
def test_rows_of_one_label_and_two(gpu, dt, codes):
    """Runs of rows of one label, whose borders lie inside workgroups: tables from LDS and from memory."""
    rows, cols = 2000, 2560
    x, branch, kw, table, w = norm._case(rows, cols, dt, dt, True, True, True, 7, gpu)
    kw['labels'] = (torch.arange(rows) // 333).int().to(gpu)
    r = block_norm.residual_norm(x, branch, weight=w, eps=1e-7, **kw, **table, quantize=codes, want_normalized=True)
    assert_close(r['x'], *norm.residual_update(x, branch, **kw), 'updated rows')
    want = kernels.norm_quantize(r['x'], w, table['shift'], table['scale'], kw['labels'], eps=1e-7, quantize=codes,
                                 want_normalized=True)
    for key in want:
        assert torch.equal(r[key], want[key]), key


@pytest.mark.parametrize('n,dtype,zeros,bias,residual', [(77, F16, True, True, True), (130, BF16, False, False, True),
                                                         (96, BF16, True, True, False)])
@pytest.mark.parametrize('k,group', [(8224, 32), (8256, 64), (8320, 128), (8448, 256), (14336, 128)])
@pytest.mark.parametrize('m', [1, 5, 8])
def test_few_rows_of_long_sums(gpu, m, k, group, n, dtype, zeros, bias, residual):
    # 257, 129, 65, 66 and 112 blocks over eight waves in pairs: a last turn that is ragged, and one that is not.
    w4.test_linear_w4(gpu, m, n, k, group, dtype, zeros, bias, residual, False)


@pytest.mark.parametrize('m,n,k,group,dtype', [(4, 66, 8320, 128, F16), (1, 200, 14336, 128, BF16)])
def test_few_gated_rows_of_long_sums(gpu, m, n, k, group, dtype):
    w4.test_linear_w4(gpu, m, n, k, group, dtype, True, True, False, True)


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('m', [1, 8, 20, 64, 200])
@pytest.mark.parametrize('k,group', [(1024, 128), (8320, 64)])
def test_inputs_of_one_sign(gpu, m, k, group, dtype):
    """All of x positive: sums of (16 + c) x and of x grow with k where the result does
    not, which the bound counts by sums of sizes."""
    codes, s = w4._case(m, 150, k, group, dtype, m % 2 == 0, False, False, gpu)
    s['x'] = (s['x'].float().abs() + 1).to(dtype)
    codes[2] = 8                                # (with zeros of 8 a row of no weight)
    y = w4._call(codes, s)
    assert_close(y, *exact_w4(s['x'], codes, s['scales'], s['zeros']), 'outputs')


def test_equal_calls_give_equal_bits(gpu):
    """On new inputs, after other calls, and again."""
    x, branch, kw, table, w = norm._case(6814, 1280, F16, F32, False, True, True, 3, gpu)
    codes, s = w4._case(70, 640, 2048, 128, BF16, True, True, True, gpu)

    def run():
        r = block_norm.residual_norm(x, branch, weight=w, eps=1e-7, **kw, **table, quantize=True)
        return [r['x'], r['q'], r['scale'], w4._call(codes, s)]
    first = run()
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(run(), first))
