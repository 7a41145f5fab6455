"""The operators around a block's projections together, as a text-encoder block
runs them: residual update and norm, 4-bit QKV projection, rotary positions in
place on the packed rows, attention, 4-bit output projection, the next update,
and the gated 4-bit feed-forward. Every stage against its 64-bit statement on
the stage's own inputs; then the whole chain captured, replayed and run on
another stream, bit for bit."""
import pytest
import torch

from block_refs import assert_close, linear_w4 as exact_w4, residual_update, rope
from w8a8 import axial_rope, block_norm, kernels, linear_w4

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, FFN = 512, 4, 768


def _weights(gpu):
    g = torch.Generator().manual_seed(11)

    def linear(n, k, **kw):
        mod = linear_w4.LinearW4(k, n, device=gpu, **kw)
        return mod.load_weight((torch.randn((n, k), generator=g) * 0.04).to(gpu))
    w = dict(qkv=linear(3 * HEADS * 128, HIDDEN), out=linear(HIDDEN, HEADS * 128, zeros=True, group_size=64),
             gate_up=linear(2 * FFN, HIDDEN, gated=True), down=linear(HIDDEN, FFN, group_size=256))
    for name in ('norm1', 'post1', 'norm2', 'post2', 'q_gain', 'k_gain'):
        n = 128 if name.endswith('gain') else HIDDEN
        w[name] = (torch.rand(n, generator=g) + 0.5).to(gpu)
    w['inv'], w['axis'] = axial_rope.ladder((24, 20, 20), shared=True, interleaved=True, device=gpu)
    return w


def _chain(w, x, branch, pos, keep=None):
    keep = {} if keep is None else keep
    rows = x.shape[0]
    a = keep['a'] = block_norm.residual_norm(x, branch, weight=w['norm1'], eps=1e-6, post_weight=w['post1'],
                                             post_eps=1e-6)
    packed = w['qkv'](a['y'])
    keep['packed'] = packed.clone()
    q, k, v = (t.unflatten(1, (HEADS, 128)) for t in packed.split(HEADS * 128, 1))
    axial_rope.rotate(q, k, pos, w['inv'], w['axis'], q_gain=w['q_gain'], k_gain=w['k_gain'], out=(q, k))
    keep['q'], keep['k'] = q, k
    prep = kernels.attention_prepare(*(t.transpose(0, 1)[None] for t in (q, k, v)))
    attn = torch.empty((rows, HEADS, 128), dtype=torch.float16, device=x.device)
    kernels.attention(prep, out=attn.transpose(0, 1)[None])
    keep['attn'] = attn.view(rows, -1)
    keep['o'] = w['out'](keep['attn'])
    b = keep['b'] = block_norm.residual_norm(a['x'], keep['o'], weight=w['norm2'], eps=1e-6, post_weight=w['post2'],
                                             post_eps=1e-6, residual_scale=0.5, branch_scale=0.25)
    keep['h'] = w['gate_up'](b['y'])
    keep['y'] = w['down'](keep['h'], residual=b['x'])
    return keep['y']


def _inputs(rows, gpu, seed=0):
    g = torch.Generator().manual_seed(rows + seed)
    return ((torch.randn((rows, HIDDEN), generator=g) * 0.3).half().to(gpu),
            torch.randn((rows, HIDDEN), generator=g).half().to(gpu),
            torch.randint(0, 3000, (rows, 3), generator=g).to(gpu))


def _check_w4(mod, x, y, residual=None, **kw):
    exact, slack = exact_w4(x, linear_w4.unpack(mod.codes), mod.scales, mod.zeros, residual=residual, gated=mod.gated)
    assert_close(y, exact, slack, **kw)


@pytest.mark.parametrize('rows', [1, 17, 130, 1000])
def test_stages(gpu, rows):
    w = _weights(gpu)
    x, branch, pos = _inputs(rows, gpu)
    s = {}
    _chain(w, x, branch, pos, s)
    torch.cuda.synchronize()
    assert_close(s['a']['x'], *residual_update(x, branch, post_weight=w['post1'], post_eps=1e-6), 'first update')
    _check_w4(w['qkv'], s['a']['y'], s['packed'], what='qkv')
    for i, (n, gain) in enumerate((('q', 'q_gain'), ('k', 'k_gain'))):
        before = s['packed'][:, i * HEADS * 128:(i + 1) * HEADS * 128].unflatten(1, (HEADS, 128))
        assert_close(s[n], *rope(before, pos, w['inv'], w['axis'], gain=w[gain]), n)
    _check_w4(w['out'], s['attn'], s['o'], what='out')
    assert_close(s['b']['x'], *residual_update(s['a']['x'], s['o'], post_weight=w['post2'], post_eps=1e-6,
                                               residual_scale=0.5, branch_scale=0.25), 'second update')
    _check_w4(w['gate_up'], s['b']['y'], s['h'], what='gate and up')
    _check_w4(w['down'], s['h'], s['y'], residual=s['b']['x'], what='down')


@pytest.mark.parametrize('rows', [1, 60, 400])
def test_captured_and_on_another_stream(gpu, rows):
    w = _weights(gpu)
    sets = [_inputs(rows, gpu, seed) for seed in range(3)]
    eager = [_chain(w, *s).clone() for s in sets]
    held = [t.clone() for t in sets[0]]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        for s, want in zip(sets, eager):
            got = _chain(w, *s)
            stream.synchronize()
            assert torch.equal(got, want)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = _chain(w, *held)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    for rep in range(4):
        for s, want in zip(sets, eager):
            for t, v in zip(held, s):
                t.copy_(v)
            out.fill_(0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), rep
            assert torch.equal(_chain(w, *s), want), rep       # eager work between the replays
            torch.cuda.synchronize()


def test_two_streams_at_once(gpu):
    """Calls that overlap on two streams share nothing."""
    w = _weights(gpu)
    sets = [_inputs(rows, gpu) for rows in (3, 500)]
    want = [_chain(w, *s).clone() for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append([_chain(w, *s) for _ in range(3)])
        torch.cuda.synchronize()
        for outs, v in zip(got, want):
            assert all(torch.equal(o, v) for o in outs)


def test_host_routes_agree(gpu):
    """The native calls and the Python wrappers make the same call."""
    w = _weights(gpu)
    x, branch, pos = _inputs(37, gpu)
    gate = torch.randn((3, HIDDEN), device=gpu)
    labels = (torch.arange(37, device=gpu) % 3).int()
    for kw in (dict(), dict(eps=1e-6), dict(eps=1e-6, weight=w['norm1'], quantize=True, post_eps=1e-5),
               dict(eps=1e-6, gate=gate, labels=labels, shift=gate, scale=gate, quantize=True, want_normalized=True,
                    convrot=False, residual_scale=2, branch_scale=0.5),
               dict(eps=1e-6, quantize=True, round_rotated=False, post_eps=1e-5, post_weight=w['post1'])):
        for b in (branch, branch.float()):
            one, two = block_norm.residual_norm(x, b, **kw), kernels.residual_norm(x, b, **kw)
            assert one.keys() == two.keys()
            for key in one:
                assert torch.equal(one[key], two[key]) and one[key].shape == two[key].shape, (kw.keys(), key)
    q = torch.randn((37, 6, 128), device=gpu).half()
    k = torch.randn((37, 2, 128), device=gpu).half()
    for args, kw in (((q, k), {}), ((q, None), dict(q_gain=w['q_gain'])),
                     ((q, k), dict(q_gain=w['q_gain'], k_gain=w['k_gain']))):
        one = axial_rope.rotate(*args, pos, w['inv'], w['axis'], pairing='adjacent', **kw)
        two = kernels.axial_rope(*args, pos, w['inv'], w['axis'], adjacent=True, **kw)
        assert torch.equal(one[0], two[0]) and (one[1] is None) == (two[1] is None)
        assert one[1] is None or torch.equal(one[1], two[1])
    m = w['out']
    a = torch.randn((3, 7, HEADS * 128), device=gpu).half()
    r = torch.randn((3, 7, HIDDEN), device=gpu).half()
    assert torch.equal(linear_w4.linear(a, m.codes, m.scales, m.zeros, residual=r),
                       kernels.linear_w4(a, m.codes, m.scales, m.zeros, residual=r))
