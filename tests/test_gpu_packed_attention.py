"""Attention of packed sequences against 64 bits (tolerances: attention_refs)."""
import math

import pytest
import torch

from attention_refs import attention64, bound, check, check_packed, starts_of
from w8a8 import _abi
from w8a8.packed_attention import packed_attention

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def make(dtype, rows, keys, heads, kv, dim, seed=0, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn((rows, heads, dim), generator=g) * scale).to(dtype).cuda()
    k = torch.randn((keys, kv, dim), generator=g).to(dtype).cuda()
    v = torch.randn((keys, kv, dim), generator=g).to(dtype).cuda()
    return q, k, v


def run(dtype, heads, kv, dim, new, keys, causal, seed=0):
    st, starts = starts_of(new, 'cuda')
    ks, k_starts = starts_of(keys, 'cuda')
    q, k, v = make(dtype, st[-1], ks[-1], heads, kv, dim, seed)
    y = packed_attention(q, k, v, starts, k_starts, causal=causal)
    check_packed(y, q, k, v, st, ks, causal, dim ** -0.5)


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('dim', [8, 24, 64, 72, 80, 96, 104, 128, 136, 256])
@pytest.mark.parametrize('dtype', DTYPES)
def test_dims(gpu, dtype, dim, causal):
    run(dtype, 4, 2, dim, [70, 1, 33], [70, 1, 65], causal, seed=dim)


LENGTHS = [([1], [1]), ([1], [300]), ([31], [31]), ([32, 33], [32, 33]), ([127, 128, 129], [127, 128, 129]),
           ([353], [353]), ([5, 0, 7], [5, 0, 7]), ([0, 0, 3, 0], [0, 4, 9, 2]), ([63, 64, 65], [64, 65, 127]),
           ([200, 3, 2], [30, 0, 5]), ([17] * 70, [19] * 70), ([257], [700])]


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('new,keys', LENGTHS)
def test_lengths(gpu, new, keys, causal):
    run(torch.bfloat16, 2, 1, 128, new, keys, causal)
    run(torch.float16, 2, 2, 64, new, keys, causal)


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('dtype,dim', [(torch.bfloat16, 128), (torch.float16, 72), (torch.bfloat16, 64), (torch.float16, 200)])
@pytest.mark.parametrize('new,keys', [([16], [4000]), ([1, 1, 1], [3000, 1, 2900]), ([130], [3001]), ([300, 2], [40, 5000]),
                                      ([0, 7, 33], [900, 2500, 2600])])
def test_few_rows_behind_many_keys(gpu, new, keys, dtype, dim, causal):
    """Workgroups share a tile's keys and join their sums."""
    shared = _abi.load().w8a8_packed_attention_workspace_size(sum(new), sum(keys), len(new), 4, 2, dim) > 0
    assert shared or len(new) > 1
    run(dtype, 4, 2, dim, new, keys, causal, seed=dim)


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('dim', [64, 72, 128, 200])
@pytest.mark.parametrize('dtype', DTYPES)
def test_more_tiles_than_compute_units(gpu, dtype, dim, causal):
    """A workgroup takes a tile with all of its keys."""
    run(dtype, 112, 4, dim, [300, 0, 33], [300, 5, 177], causal, seed=dim)


def test_masked_keys_of_many_tiles_have_no_effect(gpu):
    st, starts = starts_of([353], 'cuda')
    q, k, v = make(torch.float16, 353, 353, 112, 4, 128, seed=9)
    clean = packed_attention(q, k, v, starts)
    vv, kk = v.clone(), k.clone()
    vv[200, 1::2, ::3], kk[200, 1::2, 1::4] = math.inf, math.nan
    y = packed_attention(q, kk, vv, starts)
    assert torch.equal(y[:200], clean[:200])
    assert torch.equal(y[:, :28], clean[:, :28]) and bool(torch.isnan(y[200:, 28:56, ::3]).all())


def test_shared_keys_that_are_masked_have_no_effect(gpu):
    st, starts = starts_of([40], 'cuda')
    ks, k_starts = starts_of([3000], 'cuda')
    q, k, v = make(torch.bfloat16, 40, 3000, 2, 1, 128, seed=9)
    vv, kk = v.clone(), k.clone()
    vv[2980, :, ::3], kk[2980, :, 1::4] = math.nan, math.inf
    y = packed_attention(q, kk, vv, starts, k_starts)
    check_packed(y[:20], q[:20], k[:2980], v[:2980], [0, 20], [0, 2980], True, 128 ** -0.5)
    assert bool(torch.isnan(y[20:, :, ::3]).all())
    out = torch.full((50, 2, 128), 5.0, dtype=torch.bfloat16, device='cuda')
    q = torch.cat([q, q[:10]])
    packed_attention(q, k, v, starts, k_starts, out=out)
    check_packed(out, q, k, v, st, ks, True, 128 ** -0.5)
    assert bool((out[40:] == 5.0).all())
    fresh = packed_attention(q, k, v, starts, k_starts)
    assert torch.equal(fresh[:40], out[:40]) and not bool(fresh[40:].any())


def test_more_sequences_than_lanes(gpu):
    """Tiles are found 64 sequences at a time."""
    new = [(7 * i) % 150 for i in range(131)]
    run(torch.float16, 1, 1, 64, new, [n + 3 * (i % 40) for i, n in enumerate(new)], True)


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('sequences', [7, 8, 9, 63, 64, 65, 700, 4200])
def test_many_sequences(gpu, sequences, causal):
    """Empty ones among them, and rows behind the last."""
    g = torch.Generator().manual_seed(sequences)
    new = (torch.randint(0, 90, (sequences,), generator=g) if sequences < 100 else
           torch.randint(0, 7, (sequences,), generator=g)).tolist()
    new[1] = new[sequences // 2] = new[-1] = 0
    keys = [n + i % 3 for i, n in enumerate(new)]
    st, starts = starts_of(new, 'cuda')
    ks, k_starts = starts_of(keys, 'cuda')
    q, k, v = make(torch.bfloat16, st[-1] + 200, ks[-1], 3, 1, 16, seed=sequences)
    out = torch.full_like(q, 5.0)
    packed_attention(q, k, v, starts, k_starts, causal=causal, out=out)
    check_packed(out, q, k, v, st, ks, causal, 0.25)
    assert bool((out[st[-1]:] == 5.0).all())
    fresh = packed_attention(q, k, v, starts, k_starts, causal=causal)
    assert torch.equal(fresh[:st[-1]], out[:st[-1]]) and not bool(fresh[st[-1]:].any())


@pytest.mark.parametrize('heads,kv', [(1, 1), (6, 2), (8, 1), (20, 1), (7, 7), (64, 8)])
def test_grouped_heads(gpu, heads, kv):
    run(torch.float16, heads, kv, 128, [40, 100], [40, 120], True)


@pytest.mark.parametrize('dim', [64, 96, 128, 256])
def test_sharp_softmax(gpu, dim):
    # Scores of some hundreds: a running maximum that rises late, and rows of one key.
    st, starts = starts_of([150], 'cuda')
    q, k, v = make(torch.bfloat16, 150, 150, 2, 1, dim, seed=3, scale=12.0)
    k[100] *= 8
    y = packed_attention(q, k, v, starts)
    check_packed(y, q, k, v, st, st, True, dim ** -0.5)
    y = packed_attention(q, k, v, starts, causal=False, scale=0.01)
    check_packed(y, q, k, v, st, st, False, 0.01)


def test_layouts(gpu):
    """Views of one packed buffer, head-major tensors, an output between others, rows off 16 bytes."""
    st, starts = starts_of([45, 90], 'cuda')
    g = torch.Generator().manual_seed(5)
    buf = torch.randn((135, 4 + 2 + 2, 64), generator=g).half().cuda()
    q, k, v = buf[:, :4], buf[:, 4:6], buf[:, 6:]
    want = packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), starts)
    check_packed(want, q, k, v, st, st, True, 0.125)
    assert torch.equal(packed_attention(q, k, v, starts), want)
    hq, hk, hv = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    assert torch.equal(packed_attention(hq, hk, hv, starts), want)
    wide = torch.zeros((135, 9, 64), dtype=torch.float16, device='cuda')
    out = wide[:, 3:7]
    assert packed_attention(q, k, v, starts, out=out) is out
    assert torch.equal(out, want) and not bool(wide[:, :3].any()) and not bool(wide[:, 7:].any())
    odd = torch.zeros(135 * 4 * 64 + 3, dtype=torch.float16, device='cuda')[3:].view(135, 4, 64)
    odd.copy_(q)
    assert torch.equal(packed_attention(odd, k, v, starts), want)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)   # channels not contiguous
    assert torch.equal(packed_attention(turned, k, v, starts), want)
    one = k[:, :1].expand(135, 4, 64)                         # a broadcast key head
    assert torch.equal(packed_attention(q, one, v[:, :1].expand(135, 4, 64), starts),
                       packed_attention(q, k[:, :1], v[:, :1], starts))


def test_rows_behind_the_last_sequence(gpu):
    st, starts = starts_of([130, 20], 'cuda')
    q, k, v = make(torch.bfloat16, 300, 310, 4, 2, 128)
    q[150:], k[150:], v[150:] = math.nan, math.nan, math.inf
    y = packed_attention(q, k, v, starts, starts)
    check_packed(y, q, k, v, st, st, True, 128 ** -0.5)
    assert not bool(y[150:].any())
    out = torch.full_like(q, 7.0)
    packed_attention(q, k, v, starts, starts, out=out)
    assert torch.equal(out[:150], y[:150]) and bool((out[150:] == 7.0).all())


@pytest.mark.parametrize('bad', [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize('dim', [64, 128, 256])
def test_masked_keys_have_no_effect(gpu, dim, bad):
    """Infinities and NaNs in keys and values that a query does not see."""
    st, starts = starts_of([100, 60], 'cuda')
    for dtype in DTYPES:
        q, k, v = make(dtype, 160, 160, 2, 1, dim, seed=9)
        clean = packed_attention(q, k, v, starts)
        for at in (99, 75, 64):
            kk, vv = k.clone(), v.clone()
            vv[at, :, ::3] = bad
            kk[at, :, 1::4] = bad
            y = packed_attention(q, kk, vv, starts)
            check_packed(y[:at], q[:at], k[:at], v[:at], [0, at], [0, at], True, dim ** -0.5, f'before key {at}')
            assert torch.equal(y[100:], clean[100:])
            assert bool(torch.isnan(y[at:100]).any())


@pytest.mark.parametrize('bad', [math.inf, math.nan])
@pytest.mark.parametrize('dim,shared', [(72, False), (72, True), (80, False), (80, True), (96, False), (40, True)])
def test_masked_keys_of_other_widths_have_no_effect(gpu, dim, shared, bad):
    """Whatever takes the sums of P, and whether or not workgroups share the keys."""
    nk = 1500 if shared else 90
    starts, k_starts = starts_of([90], 'cuda')[1], starts_of([nk], 'cuda')[1]
    assert (_abi.load().w8a8_packed_attention_workspace_size(90, nk, 1, 2, 2, dim) > 0) == shared
    for dtype in DTYPES:
        q, k, v = make(dtype, 90, nk, 2, 2, dim, seed=dim)
        at = nk - 30
        k[at, :, 1::4], v[at, :, ::3] = bad, bad
        y = packed_attention(q, k, v, starts, k_starts)
        check_packed(y[:60], q[:60], k[:at], v[:at], [0, 60], [0, at], True, dim ** -0.5)
        assert bool(torch.isnan(y[60:, :, ::3]).all())


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('dtype,dim', [(torch.bfloat16, 128), (torch.float16, 80), (torch.bfloat16, 256)])
@pytest.mark.parametrize('sequences', [8, 40, 70])
def test_few_rows_of_many_sequences(gpu, sequences, dtype, dim, causal):
    """Sequences are searched for, and workgroups share their keys."""
    g = torch.Generator().manual_seed(sequences)
    new = torch.randint(0, 4, (sequences,), generator=g).tolist()
    keys = (torch.randint(500, 900, (sequences,), generator=g) if sequences < 70 else
            torch.randint(0, 1800, (sequences,), generator=g)).tolist()
    new[0], keys[-1], new[-1] = 0, 0, 2
    assert _abi.load().w8a8_packed_attention_workspace_size(sum(new), sum(keys), sequences, 2, 1, dim) > 0
    run(dtype, 2, 1, dim, new, keys, causal, seed=dim)


def test_visible_infinities(gpu):
    _, starts = starts_of([70], 'cuda')
    q, k, v = make(torch.bfloat16, 70, 70, 1, 1, 64)
    v[10, 0, 5], v[66, 0, 6], v[67, 0, 6], v[68, 0, 7] = math.inf, math.inf, -math.inf, math.nan
    y = packed_attention(q, k, v, starts)[:, 0]
    assert bool((y[10:, 5] == math.inf).all()) and bool(torch.isfinite(y[:10]).all())
    assert bool(torch.isfinite(y[:66, 6]).all()) and float(y[66, 6]) == math.inf
    assert bool(torch.isnan(y[67:, 6]).all())
    assert bool(torch.isfinite(y[:68, 7]).all()) and bool(torch.isnan(y[68:, 7]).all())
    assert bool(torch.isfinite(y[:, 8:]).all())


def test_far_rows(gpu):
    """Keys whose offsets pass 32 bits."""
    rows, stride = 600, 1 << 22
    big = torch.empty(rows * stride, dtype=torch.float16, device='cuda').view(rows, 1, stride)
    k, v = big[:, :, :64], big[:, :, 64:128]
    q, kk, vv = make(torch.float16, 200, rows, 1, 1, 64)
    k.copy_(kk)
    v.copy_(vv)
    st, starts = starts_of([200], 'cuda')
    ks, k_starts = starts_of([rows], 'cuda')
    y = packed_attention(q, k, v, starts, k_starts)
    check_packed(y, q, kk, vv, st, ks, True, 0.125)


def test_long_sequence(gpu):
    st, starts = starts_of([5, 4099], 'cuda')
    q, k, v = make(torch.bfloat16, 4104, 4104, 2, 1, 128)
    y = packed_attention(q, k, v, starts)
    check_packed(y, q, k, v, st, st, True, 128 ** -0.5)
    assert torch.equal(packed_attention(q, k, v, starts), y)   # the same bits every time


def test_captured_and_on_another_stream(gpu):
    """A graph replayed over other contents, lengths and starts; two streams at once."""
    q, k, v = make(torch.bfloat16, 300, 300, 4, 2, 128)
    starts = torch.tensor([0, 100, 300], dtype=torch.int32, device='cuda')
    out = torch.empty_like(q)
    packed_attention(q, k, v, starts, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            packed_attention(q, k, v, starts, out=out)
    torch.cuda.current_stream().wait_stream(side)
    for seed, cut in ((1, 100), (2, 7), (3, 300), (4, 0)):
        q2, k2, v2 = make(torch.bfloat16, 300, 300, 4, 2, 128, seed=seed)
        for t, s in ((q, q2), (k, k2), (v, v2)):
            t.copy_(s)
        starts.copy_(torch.tensor([0, cut, 300], dtype=torch.int32))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check_packed(out, q2, k2, v2, [0, cut, 300], [0, cut, 300], True, 128 ** -0.5)
        with torch.cuda.stream(side):
            other = packed_attention(q2, k2, v2, starts)
        here = packed_attention(q2, k2, v2, starts)
        torch.cuda.synchronize()
        assert torch.equal(other, out) and torch.equal(here, out)


def test_starts_out_of_range_stay_in_bounds(gpu):
    """Starts beyond the rows are cut off at the rows."""
    q, k, v = make(torch.float16, 50, 50, 2, 1, 64)
    starts = torch.tensor([0, 30, 90], dtype=torch.int32, device='cuda')
    y = packed_attention(q, k, v, starts)
    check_packed(y, q, k, v, [0, 30, 50], [0, 30, 50], True, 0.125)


def test_no_rows_and_no_keys(gpu):
    starts = torch.zeros(3, dtype=torch.int32, device='cuda')
    q, k, v = make(torch.float16, 0, 0, 2, 1, 64)
    assert packed_attention(q, k, v, starts).shape == (0, 2, 64)
    q, _, _ = make(torch.float16, 40, 0, 2, 1, 64)
    st = torch.tensor([0, 10, 40], dtype=torch.int32, device='cuda')
    assert not bool(packed_attention(q, k, v, st, starts).any())


def test_differentiable_inputs_are_refused(gpu):
    q, k, v = make(torch.float16, 8, 8, 1, 1, 64)
    starts = torch.tensor([0, 8], dtype=torch.int32, device='cuda')
    with pytest.raises(ValueError, match='no gradient'):
        packed_attention(q.requires_grad_(), k, v, starts)
    with torch.no_grad():
        packed_attention(q, k, v, starts)


def test_reference_matches_its_bound(gpu):
    """The bound holds for the plain form in the operands' type too."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn((64, 64), generator=g).bfloat16() for _ in range(3))
    o, parts = attention64(q.double(), k.double(), v.double(), 0.125)
    p = torch.exp((q.float() @ k.float().t()) * 0.125 - ((q.float() @ k.float().t()) * 0.125).amax(1, keepdim=True))
    y = ((p.bfloat16().float() @ v.float()) / p.sum(1, keepdim=True)).bfloat16()
    check(y, o, bound(o, parts, torch.bfloat16))
