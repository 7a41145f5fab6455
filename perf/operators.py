"""Performance cases of the operators around the projections of a block.

Three operators, as a DiT or text-encoder step calls them:

  norm    the update of the residual stream by a block's branch (its own RMS
          norm, AdaLN gate and scales) with the next block's RMS norm and
          modulation, to normalized rows or to ConvRot256 INT8 codes
  rope    per-head RMS norm and rotary positions of several axes for Q and K
  w4      projections with 4-bit weights and group scales, plain and gated

``own`` false computes them from elementary torch operations in 32 bits
(angles in 64), true through the package. ``prepare`` makes the same inputs
for both.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {'f16': torch.float16, 'bf16': torch.bfloat16, 'f32': torch.float32}
MOD_ROWS = 9        # AdaLN table rows of one DiT forward
DIVISOR = 512.0     # residual divisor of the scaled FP16 tensor flow


def listed():
    return [
        # One decode token of the text encoder between two blocks: latency.
        dict(name='norm_token', op='norm', m=1, k=5120, dtype='f16', branch='f16', post=False, gate=False, mod=False,
             quant=False),
        # A 353-token prompt through a sandwich-norm block (norm after the block and before the next).
        dict(name='norm_prompt_sandwich', op='norm', m=353, k=5120, dtype='bf16', branch='bf16', post=True, gate=False,
             mod=False, quant=False),
        # A DiT request after the exchange of rank partials (FP32 branch), to the next projection's INT8 codes.
        dict(name='norm_dit_codes', op='norm', m=6814, k=5376, dtype='f16', branch='f32', post=False, gate=True,
             mod=True, quant=True),
        # A whole clip's rows: norm after the block, gate, and the next modulated norm.
        dict(name='norm_clip', op='norm', m=53504, k=5376, dtype='f16', branch='f16', post=True, gate=True, mod=True,
             quant=False),
        # One decode token, 64 query and 8 key heads, three interleaved axes far into a context: latency.
        dict(name='rope_token', op='rope', m=1, hq=64, hk=8, d=128, rot=128, axes=3, order='interleaved',
             pairing='half', dtype='f16', norm=True, far=30000),
        # A prompt with images, the same heads in bf16.
        dict(name='rope_prompt', op='rope', m=353, hq=64, hk=8, d=128, rot=128, axes=3, order='interleaved',
             pairing='half', dtype='bf16', norm=True, far=1000),
        # Patches of an image encoder: 72-wide heads, height and width, no norm, fp32.
        dict(name='rope_patches', op='rope', m=4097, hq=16, hk=16, d=72, rot=72, axes=2, order='sections',
             pairing='half', dtype='f32', norm=False, far=64),
        # A clip on one rank: 28 heads, the 96-wide rotary prefix over time, height and width.
        dict(name='rope_clip', op='rope', m=53504, hq=28, hk=28, d=128, rot=96, axes=3, order='sections',
             pairing='half', dtype='f16', norm=True, far=76),
        # One decode token through an up projection: weight streaming and latency.
        dict(name='w4_token', op='w4', m=1, n=14336, k=4096, group=128, dtype='f16', zeros=False, gated=False,
             bias=False, residual=False),
        # A short prompt (64 rows) through a down projection with zero points and the residual.
        dict(name='w4_short_prompt', op='w4', m=64, n=4096, k=14336, group=128, dtype='bf16', zeros=True, gated=False,
             bias=False, residual=True),
        # A 353-token prompt through gate and up of the text encoder.
        dict(name='w4_gated_prompt', op='w4', m=353, n=25600, k=5120, group=128, dtype='f16', zeros=False, gated=True,
             bias=False, residual=False),
        # A long prompt with a fine scale grid and a bias.
        dict(name='w4_long_prompt', op='w4', m=2048, n=14336, k=4096, group=64, dtype='bf16', zeros=True, gated=False,
             bias=True, residual=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['norm', 'rope', 'w4'])
    if op == 'norm':
        quant = rng.random() < 0.4
        step = 256 if quant else 16
        k = _log(rng, 256, 8192) // step * step
        m = _log(rng, 1, min(53504, 53504 * 5376 // k))
        dtype = rng.choice(['f16', 'bf16'])
        return dict(op='norm', m=m, k=k, dtype=dtype, branch=rng.choice([dtype, dtype, 'f32']),
                    post=rng.random() < 0.5, gate=rng.random() < 0.5, mod=rng.random() < 0.5, quant=quant)
    if op == 'rope':
        d = rng.choice([64, 72, 80, 96, 128, 256])
        axes = rng.choice([1, 2, 3, 4])
        rot = d if rng.random() < 0.5 else max(2 * axes, d * rng.randint(1, 4) // 4 // 2 * 2)
        hq = rng.choice([8, 12, 16, 28, 32, 64])
        hk = rng.choice([h for h in (1, 2, 4, 8, 12, 16, 28) if hq % h == 0])
        m = _log(rng, 1, min(53504, 53504 * 56 * 128 // ((hq + hk) * d)))
        dtype = rng.choice(['f16', 'bf16', 'f32'])
        if dtype == 'f32':
            m = max(1, m // 2)
        return dict(op='rope', m=m, hq=hq, hk=hk, d=d, rot=rot, axes=axes,
                    order=rng.choice(['sections', 'interleaved']), pairing=rng.choice(['half', 'adjacent']),
                    dtype=dtype, norm=rng.random() < 0.5, far=_log(rng, 16, 1000000))
    group = rng.choice([32, 64, 128, 128, 256])
    k = max(group, _log(rng, 256, 14336) // group * group)
    gated = rng.random() < 0.4
    n = _log(rng, 128, 25600) // 2 * 2
    m = _log(rng, 1, max(1, min(2048, 2048 * 14336 * 4096 // (n * k))))
    return dict(op='w4', m=m, n=n, k=k, group=group, dtype=rng.choice(['f16', 'bf16']), zeros=rng.random() < 0.5,
                gated=gated, bias=rng.random() < 0.3, residual=not gated and rng.random() < 0.3)


# ------------------------------------------------------------------ inputs
def _labels(m):
    """AdaLN rows by frame: sixteen equal runs of rows cycling over the table."""
    frames = min(16, m)
    bounds = [m * i // frames for i in range(frames + 1)]
    return torch.cat([torch.full((bounds[i + 1] - bounds[i],), i % MOD_ROWS, dtype=torch.int32)
                      for i in range(frames)]).cuda()


def _prepare_norm(c, g):
    m, k, dt = c['m'], c['k'], DTYPES[c['dtype']]

    def rand(*shape):
        return torch.randn(shape, generator=g, device='cuda')
    x = rand(m, k).mul_(3.0 / DIVISOR)
    x[:, ::max(1, k // 8)] *= 20.0          # a few outlier channels, as residual streams have
    s = dict(x=x.to(dt), branch=rand(m, k).mul_(1.0 if c['post'] else 1.0 / DIVISOR).to(DTYPES[c['branch']]),
             weight=rand(k).mul_(0.2).add_(1.0), eps=1e-6 / DIVISOR ** 2, residual_scale=1.0, branch_scale=1.0)
    if c['post']:
        s.update(post_weight=rand(k).mul_(0.2).add_(1.0), post_eps=1e-6, branch_scale=1.0 / DIVISOR)
    if c['gate']:
        s['gate'] = rand(MOD_ROWS, k).mul_(0.5)
    if c['mod']:
        s['shift'], s['scale'] = rand(MOD_ROWS, k).mul_(0.1), rand(MOD_ROWS, k).mul_(0.1)
    if c['gate'] or c['mod']:
        s['labels'] = _labels(m)
    return s


def _prepare_rope(c, g):
    m, rot, axes, dt = c['m'], c['rot'], c['axes'], DTYPES[c['dtype']]
    half = rot // 2
    q = torch.randn((m, c['hq'], c['d']), generator=g, device='cuda').to(dt)
    k = torch.randn((m, c['hk'], c['d']), generator=g, device='cuda').to(dt)
    pos = torch.randint(0, c['far'] + 1, (m, axes), generator=g, device='cuda')
    i = torch.arange(half, dtype=torch.float64, device='cuda')
    if c['order'] == 'interleaved':         # one ladder over all pairs, the axes in turn
        inv_freq, axis = 10000.0 ** (-i / half), (torch.arange(half, device='cuda') % axes).int()
    else:                                   # a ladder of its own for each axis' run of pairs
        runs = [half // axes + (a < half % axes) for a in range(axes)]
        inv_freq = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in runs]).cuda()
        axis = torch.cat([torch.full((n,), a, dtype=torch.int32) for a, n in enumerate(runs)]).cuda()
    s = dict(q=q, k=k, positions=pos, inv_freq=inv_freq, axis=axis, q_gain=None, k_gain=None)
    if c['norm']:
        s['q_gain'] = torch.rand(c['d'], generator=g, device='cuda') + 0.5
        s['k_gain'] = torch.rand(c['d'], generator=g, device='cuda') + 0.5
    return s


def _prepare_w4(c, g):
    m, n, k, dt = c['m'], c['n'], c['k'], DTYPES[c['dtype']]
    groups = k // c['group']
    x = torch.randn((m, k), generator=g, device='cuda').mul_(0.5)
    x[:, ::max(1, k // 8)] *= 20.0
    s = dict(x=x.to(dt),
             codes=torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), generator=g, device='cuda', dtype=torch.int64).int(),
             scales=torch.rand((groups, n), generator=g, device='cuda').add_(0.5).mul_(0.004).to(dt),
             zeros=None, bias=None, residual=None)
    if c['zeros']:
        s['zeros'] = torch.randint(4, 12, (groups, n), generator=g, device='cuda').to(torch.uint8)
    if c['bias']:
        s['bias'] = torch.randn(n, generator=g, device='cuda').mul_(0.01).to(dt)
    if c['residual']:
        s['residual'] = torch.randn((m, n), generator=g, device='cuda').to(dt)
    return s


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    make = {'norm': _prepare_norm, 'rope': _prepare_rope, 'w4': _prepare_w4}[case['op']]
    return dict(make(case, g), case=case)


# ------------------------------------------------------------ plain forms
def _rotation(dtype):
    """ConvRot256 over 16: the fourth Kronecker power of the 4 x 4 matrix of
    ones whose antidiagonal is negated."""
    h4 = torch.ones((4, 4), dtype=dtype, device='cuda') - 2 * torch.eye(4, dtype=dtype, device='cuda').flip(0)
    h16 = torch.kron(h4, h4)
    return torch.kron(h16, h16) / 16


def _norm_in(s, f):
    """The operator in arithmetic of type f: the updated rows and the rows or the codes' values."""
    c = s['case']
    dt = s['x'].dtype
    b = s['branch'].to(f)
    if c['post']:
        b = b * torch.rsqrt(b.square().mean(-1, keepdim=True) + s['post_eps']) * s['post_weight'].to(f)
    b = b * s['branch_scale']
    lab = s['labels'].long() if 'labels' in s else None
    if c['gate']:
        b = b * s['gate'].to(f)[lab]
    new = (s['x'].to(f) * s['residual_scale'] + b).to(dt)
    del b
    v = new.to(f)
    y = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + s['eps']) * s['weight'].to(f)
    if c['mod']:
        y = y * (1 + s['scale'].to(f)[lab]) + s['shift'].to(f)[lab]
    if c['quant']:
        r = (y.to(dt).to(f).reshape(-1, 256) @ _rotation(f)).to(dt).to(f).reshape(y.shape)
        step = (r.abs().amax(-1, keepdim=True) / 127).clamp_min(1e-30)
        y = (r / step).round().clamp(-128, 127) * step
    return new, y


def _norm_plain(s):
    new, y = _norm_in(s, torch.float32)
    return {'x': new, 'values' if s['case']['quant'] else 'y': y.to(s['x'].dtype)}


def _angles(s):
    return s['positions'].double()[:, s['axis'].long()] * s['inv_freq']


def _turn(x, cos, sin, gain, pairing, f):
    x = x.to(f)
    if gain is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gain.to(f)
    half = cos.shape[-1]
    cos, sin = cos.to(f)[:, None], sin.to(f)[:, None]
    if pairing == 'half':
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b, rest = x[..., 0:2 * half:2], x[..., 1:2 * half:2], x[..., 2 * half:]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _rope_plain(s):
    phi = _angles(s)
    cos, sin = phi.cos(), phi.sin()
    p = s['case']['pairing']
    return {'q': _turn(s['q'], cos, sin, s['q_gain'], p, torch.float32).to(s['q'].dtype),
            'k': _turn(s['k'], cos, sin, s['k_gain'], p, torch.float32).to(s['k'].dtype)}


def _w4_plain(s):
    """A word's nibbles 0-3 hold its inputs 0, 2, 4, 6 and nibbles 4-7 its inputs 1, 3, 5, 7."""
    c = s['case']
    shifts = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device='cuda')
    w = ((s['codes'][:, :, None] >> shifts) & 15).float().reshape(c['n'], -1, c['group'])
    w = w - (s['zeros'].float().t()[:, :, None] if c['zeros'] else 8.0)
    w = (w * s['scales'].float().t()[:, :, None]).reshape(c['n'], c['k'])
    y = s['x'].float() @ w.t()
    if c['bias']:
        y = y + s['bias'].float()
    if c['gated']:
        g, u = y.chunk(2, -1)
        y = g / (1 + torch.exp(-g)) * u
    if c['residual']:
        y = y + s['residual'].float()
    return {'y': y.to(s['x'].dtype)}


# --------------------------------------------------------------- the calls
def _package():
    path = str(Path(__file__).resolve().parents[1] / 'minimax-h3-2xt4_amd')
    if path not in sys.path:
        sys.path.insert(0, path)
    from w8a8 import axial_rope, block_norm, linear_w4
    return block_norm.residual_norm, axial_rope.rotate, linear_w4.linear


_CALLS = []


def _own(s):
    if not _CALLS:
        _CALLS.extend(_package())
    c = s['case']
    if c['op'] == 'norm':
        r = _CALLS[0](s['x'], s['branch'], weight=s['weight'], eps=s['eps'], post_weight=s.get('post_weight'),
                      post_eps=s.get('post_eps'), gate=s.get('gate'), shift=s.get('shift'), scale=s.get('scale'),
                      labels=s.get('labels'), residual_scale=s['residual_scale'], branch_scale=s['branch_scale'],
                      quantize=c['quant'])
        if not c['quant']:
            return {'x': r['x'], 'y': r['y']}
        values = torch.empty_like(s['x'])
        torch.mul(r['q'], r['scale'], out=values)
        return {'x': r['x'], 'values': values}
    if c['op'] == 'rope':
        q, k = _CALLS[1](s['q'], s['k'], s['positions'], s['inv_freq'], s['axis'], pairing=c['pairing'],
                         q_gain=s['q_gain'], k_gain=s['k_gain'], eps=1e-6)
        return {'q': q, 'k': k}
    return {'y': _CALLS[2](s['x'], s['codes'], s['scales'], s['zeros'], bias=s['bias'], residual=s['residual'],
                           gated=c['gated'])}


def run(state):
    if own:
        return _own(state)
    return {'norm': _norm_plain, 'rope': _rope_plain, 'w4': _w4_plain}[state['case']['op']](state)


# ------------------------------------------------------------ exact values
def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'norm':
        parts = []
        rows = max(1, (1 << 26) // case['k'])
        for r in range(0, case['m'], rows):       # 64-bit copies of a whole clip's rows need not exist at once
            t = dict(s, x=s['x'][r:r + rows], branch=s['branch'][r:r + rows])
            if 'labels' in s:
                t['labels'] = s['labels'][r:r + rows]
            parts.append(_exact_norm(t))
        key = 'values' if case['quant'] else 'y'
        return {'x': torch.cat([p[0] for p in parts]), key: torch.cat([p[1] for p in parts])}
    if case['op'] == 'rope':
        return {n: _exact_rope(s, s[n], s[n + '_gain']) for n in ('q', 'k')}
    return {'y': _exact_w4(s)}


def _exact_norm(s):
    """In 64 bits; what the definition stores in 16 bits on the way (the updated
    and the normalized rows, the rotated ones) is rounded there, nothing else."""
    c, dt = s['case'], s['x'].dtype
    b = s['branch'].double()
    if c['post']:
        b = b / ((b * b).sum(1, keepdim=True) / c['k'] + s['post_eps']).sqrt() * s['post_weight'].double()
    b *= s['branch_scale']
    if c['gate']:
        b *= s['gate'].double().index_select(0, s['labels'])
    full = b + s['residual_scale'] * s['x'].double()
    v = full.to(dt).double()
    y = v / ((v * v).sum(1, keepdim=True) / c['k'] + s['eps']).sqrt() * s['weight'].double()
    if c['mod']:
        y = y + y * s['scale'].double().index_select(0, s['labels'])
        y += s['shift'].double().index_select(0, s['labels'])
    if not c['quant']:
        return full, y
    r = y.to(dt).double().reshape(c['k'] // 256 * v.shape[0], 4, 4, 4, 4)
    for axis in range(1, 5):                  # one factor a digit: the sum, less twice the opposite one
        r = r.sum(axis, keepdim=True) - 2 * r.flip(axis)
    r = (r / 16).to(dt).double().reshape(y.shape)
    step = r.abs().max(1, keepdim=True).values.clamp_min(127e-30) / 127
    return full, torch.clamp(torch.round(r / step), -128, 127) * step


def _exact_rope(s, x, gain):
    c = s['case']
    half = c['rot'] // 2
    v = x.double().clone()
    if gain is not None:
        v = v / ((v * v).sum(-1, keepdim=True) / c['d'] + 1e-6).sqrt() * gain.double()
    phi = torch.gather(s['positions'].double(), 1, s['axis'].long().expand(c['m'], half)) * s['inv_freq']
    first, second = ((slice(0, half), slice(half, 2 * half)) if c['pairing'] == 'half'
                     else (slice(0, 2 * half, 2), slice(1, 2 * half, 2)))
    z = torch.complex(v[..., first], v[..., second]) * torch.polar(torch.ones_like(phi), phi)[:, None]
    v[..., first], v[..., second] = z.real, z.imag
    return v


def _exact_w4(s):
    c = s['case']
    per = 8
    w = torch.empty((c['n'], c['k'] // per, per), dtype=torch.float64, device='cuda')
    for j in range(per):
        w[:, :, j] = (s['codes'] >> (4 * (j // 2) + 16 * (j % 2))) & 15
    w = w.reshape(c['n'], -1, c['group'])
    w -= s['zeros'].double().t().unsqueeze(-1) if c['zeros'] else 8
    w *= s['scales'].double().t().unsqueeze(-1)
    y = s['x'].double() @ w.reshape(c['n'], c['k']).t()
    if c['bias']:
        y += s['bias'].double()
    if c['gated']:
        y = y[:, :c['n'] // 2] * torch.sigmoid(y[:, :c['n'] // 2]) * y[:, c['n'] // 2:]
    return y + s['residual'].double() if c['residual'] else y


# ------------------------------------------------------------ needed work
def work(case):
    c, size = case, {'f16': 2, 'bf16': 2, 'f32': 4}
    e = size[c['dtype']]
    if c['op'] == 'norm':
        n = c['m'] * c['k']
        tables = MOD_ROWS * c['k'] * 4 * (c['gate'] + 2 * c['mod']) + c['k'] * 4 * (1 + c['post'])
        return {'bytes': n * (2 * e + size[c['branch']] + e) + tables + 4 * c['m'],
                'flops': n * (8 + 4 * c['post'] + 2 * c['gate'] + 3 * c['mod'] + 18 * c['quant'])}
    if c['op'] == 'rope':
        n = c['m'] * (c['hq'] + c['hk']) * c['d']
        return {'bytes': 2 * n * e + 8 * c['m'] * c['axes'] + 12 * (c['rot'] // 2) + (8 * c['d'] if c['norm'] else 0),
                'flops': n * (3 + 4 * c['norm'])}
    out = c['n'] // 2 if c['gated'] else c['n']
    groups = c['k'] // c['group']
    return {'bytes': c['n'] * c['k'] // 2 + groups * c['n'] * (e + c['zeros']) + c['m'] * c['k'] * e
            + c['m'] * out * e * (1 + c['residual']) + (c['n'] * e if c['bias'] else 0),
            'flops': 2 * c['m'] * c['n'] * c['k']}
