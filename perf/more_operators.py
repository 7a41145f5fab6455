"""Performance cases of the attention of text and image encoders.

Three operators, as a prompt and the tokens after it run through them:

  cache   keys and values written into a paged cache, 16-bit or as INT8 codes
          with a scale per token and head, and whole sequences read back
  attend  one new token of every sequence over its cached keys
  packed  attention of packed sequences of different lengths, causal or not

``own`` false computes them from elementary torch operations in 32 bits, true
through the package. ``prepare`` makes the same inputs for both.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {'f16': torch.float16, 'bf16': torch.bfloat16}


def listed():
    return [
        # One decode step of one sequence: its token's keys and values into 16-bit pages. Latency.
        dict(name='cache_token', op='cache', dtype='f16', codes=False, page=16, kv=8, dim=128, seqs=1, new=1, prefix=352,
             ragged=False, read=False),
        # The prompt of the text encoder, kept as codes and read back for the attention of what follows.
        dict(name='cache_prompt_codes', op='cache', dtype='bf16', codes=True, page=64, kv=8, dim=128, seqs=1, new=353,
             prefix=0, ragged=False, read=True),
        # Requests of many lengths arriving together, 28 heads, into 16-bit pages.
        dict(name='cache_requests', op='cache', dtype='f16', codes=False, page=64, kv=28, dim=128, seqs=12, new=1001,
             prefix=0, ragged=True, read=False),
        # The last chunk of long contexts as codes, and the contexts read back.
        dict(name='cache_contexts_codes', op='cache', dtype='bf16', codes=True, page=64, kv=8, dim=128, seqs=8, new=1024,
             prefix=7168, ragged=True, read=True),
        # One decode token behind a 353-token prompt: latency.
        dict(name='attend_token', op='attend', dtype='f16', codes=False, page=16, heads=64, kv=8, dim=128, seqs=1,
             keys=354, ragged=False),
        # A batch with 80-wide heads that share nothing, pages of 48 tokens, odd lengths.
        dict(name='attend_batch_odd', op='attend', dtype='f16', codes=False, page=48, heads=28, kv=28, dim=80, seqs=7,
             keys=1501, ragged=True),
        # A serving batch of ragged contexts in INT8 pages.
        dict(name='attend_batch_codes', op='attend', dtype='bf16', codes=True, page=64, heads=64, kv=8, dim=128, seqs=64,
             keys=4096, ragged=True),
        # One token at the end of a very long context.
        dict(name='attend_long', op='attend', dtype='bf16', codes=False, page=64, heads=64, kv=8, dim=128, seqs=1,
             keys=131072, ragged=False),
        # The 353-token prompt of the text encoder.
        dict(name='packed_prompt', op='packed', dtype='bf16', heads=64, kv=8, dim=128, seqs=1, new=353, prefix=0,
             ragged=False, causal=True),
        # Patches of an image encoder: 72-wide heads, images of different sizes, not causal.
        dict(name='packed_patches', op='packed', dtype='f16', heads=16, kv=16, dim=72, seqs=5, new=4097, prefix=0,
             ragged=True, causal=False),
        # Chunks of several prompts behind what they have cached.
        dict(name='packed_chunks', op='packed', dtype='f16', heads=64, kv=8, dim=128, seqs=6, new=500, prefix=3500,
             ragged=True, causal=True),
        # A long document.
        dict(name='packed_document', op='packed', dtype='bf16', heads=64, kv=8, dim=128, seqs=1, new=16384, prefix=0,
             ragged=False, causal=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    op = rng.choice(['cache', 'attend', 'packed'])
    dim = rng.choice([64, 72, 80, 96, 128, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 16, 28])
    group = rng.choice([g for g in (1, 2, 4, 7, 8, 16) if g * kv <= 64])
    c = dict(op=op, dtype=rng.choice(['f16', 'bf16']), kv=kv, dim=dim, ragged=rng.random() < 0.7)
    if op == 'cache':
        c.update(codes=rng.random() < 0.5, page=rng.choice([16, 32, 48, 64, 128, 256]), seqs=_log(rng, 1, 128))
        c['read'] = c['codes'] or rng.random() < 0.3
        most = 60000 * 8 * 128 // (2 * kv * dim * c['seqs'])
        c['new'] = _log(rng, 1, min(8192, max(1, most)))
        c['prefix'] = 0 if rng.random() < 0.3 else _log(rng, 1, min(32768, max(1, most)))
        return c
    c['heads'] = kv * group
    if op == 'attend':
        c.update(codes=rng.random() < 0.5, page=rng.choice([16, 32, 48, 64, 128, 256]), seqs=_log(rng, 1, 128))
        c['keys'] = _log(rng, 1, min(131072, 131072 * 8 * 128 * 3 // (4 * kv * dim * c['seqs'])))
        return c
    c.update(seqs=_log(rng, 1, 32), causal=rng.random() < 0.7)
    pairs = 16384 * 16384 * 64 * 128 // (4 * c['heads'] * dim * c['seqs'])     # of one sequence, at most
    c['new'] = _log(rng, 1, min(16384, math.isqrt(pairs)))
    c['prefix'] = 0 if rng.random() < 0.5 else _log(rng, 1, min(16384, max(1, pairs // c['new'] - c['new'])))
    return c


# ------------------------------------------------------------------ inputs
def _lengths(n, seqs, ragged):
    """Lengths of seqs sequences around n: equal, or from a quarter of n to 1.75 n."""
    if not ragged:
        return [n] * seqs
    return [max(1, int(n * (0.25 + 1.5 * ((i * 0.6180339887 + 0.5) % 1.0)))) for i in range(seqs)]


def _rows(c):
    """(new rows, keys) of every sequence."""
    if c['op'] == 'attend':
        keys = _lengths(c['keys'], c['seqs'], c['ragged'])
        return [1] * len(keys), keys
    new = _lengths(c['new'], c['seqs'], c['ragged'])
    before = _lengths(c['prefix'], c['seqs'], c['ragged']) if c['prefix'] else [0] * c['seqs']
    return new, [n + b for n, b in zip(new, before)]


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32)


def _keys(shape, g, dt):
    """Keys as they come from a norm and rotary positions: a few strong channels."""
    x = torch.randn(shape, generator=g, device='cuda')
    x[..., ::max(1, shape[-1] // 4)] *= 3.0
    return x.to(dt)


def _values(shape, g, dt):
    return torch.randn(shape, generator=g, device='cuda').mul_(0.5).to(dt)


def _pages(c, keys, g):
    """Pages of the sequences in an order that an allocator in use gives, and a cache with a few to spare."""
    need = [-(-n // c['page']) for n in keys]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device='cuda').cpu()
    table = torch.zeros((c['seqs'], max(need)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return pages, table.cuda()


def _fill(c, pages, g, dt):
    """Cache buffers [pages, heads, page, dim] with what earlier steps left in them."""
    shape = (pages, c['kv'], c['page'], c['dim'])
    k, v = _keys(shape, g, dt), _values(shape, g, dt)
    if not c['codes']:
        return dict(k=k, v=v, k_scale=None, v_scale=None)
    kq, ks = _quantize(k)
    vq, vs = _quantize(v)
    return dict(k=kq, v=vq, k_scale=ks, v_scale=vs)


def prepare(case, seed):
    c, dt = case, DTYPES[case['dtype']]
    g = torch.Generator(device='cuda').manual_seed(seed)
    new, keys = _rows(c)
    rows, total = sum(new), sum(keys)
    s = dict(case=c, new=new, keys=keys, lengths=torch.tensor(keys, dtype=torch.int32).cuda(),
             starts=_starts(new).cuda(), k_starts=_starts(keys).cuda())
    if c['op'] == 'packed':
        s.update(q=torch.randn((rows, c['heads'], c['dim']), generator=g, device='cuda').mul_(1.5).to(dt),
                 k=_keys((total, c['kv'], c['dim']), g, dt), v=_values((total, c['kv'], c['dim']), g, dt))
        return s
    pages, s['table'] = _pages(c, keys, g)
    s['cache'] = _fill(c, pages, g, dt)
    if c['op'] == 'attend':
        s['q'] = torch.randn((c['seqs'], c['heads'], c['dim']), generator=g, device='cuda').mul_(1.5).to(dt)
    else:
        s.update(k=_keys((rows, c['kv'], c['dim']), g, dt), v=_values((rows, c['kv'], c['dim']), g, dt))
    if own:
        s['handle'] = _package()[0].KVCache(**s['cache'])
    return s


# ------------------------------------------------------------ plain forms
def _quantize(x):
    """INT8 codes of the last dimension and their fp32 scale."""
    f = x.float()
    scale = (f.abs().amax(-1) * torch.tensor(1.0 / 127.0, dtype=torch.float32, device='cuda')).clamp_min(1e-30)
    return (f / scale[..., None]).round().clamp(-128, 127).to(torch.int8), scale


def _places(s):
    """(page, offset) of every new row."""
    c = s['case']
    seq = torch.repeat_interleave(torch.arange(c['seqs'], device='cuda'), s['starts'].diff().long(),
                                  output_size=sum(s['new']))
    pos = torch.arange(sum(s['new']), device='cuda') - s['starts'].long()[seq + 1] + s['lengths'].long()[seq]
    return s['table'].long()[seq, pos // c['page']], pos % c['page']


def _cache_plain(s):
    c, cache = s['case'], s['cache']
    page, off = _places(s)
    for n in ('k', 'v'):
        if c['codes']:
            cache[n][page, :, off], cache[n + '_scale'][page, :, off] = _quantize(s[n])
        else:
            cache[n][page, :, off] = s[n]
    if not c['read']:
        return {'k': cache['k'], 'v': cache['v']}
    seq = torch.repeat_interleave(torch.arange(c['seqs'], device='cuda'), s['lengths'].long(), output_size=sum(s['keys']))
    pos = torch.arange(sum(s['keys']), device='cuda') - s['k_starts'].long()[seq]
    page, off = s['table'].long()[seq, pos // c['page']], pos % c['page']
    out = {}
    for n in ('k', 'v'):
        x = cache[n][page, :, off]
        if c['codes']:
            x = (x.float() * cache[n + '_scale'][page, :, off][..., None]).to(s[n].dtype)
        out[n] = x
    return out


def _attend_plain(s):
    c, cache = s['case'], s['cache']
    table = s['table'].long()
    span = table.shape[1] * c['page']

    def whole(n):                             # [seqs, kv, keys, dim]
        x = cache[n][table].float()
        if c['codes']:
            x = x * cache[n + '_scale'][table][..., None]
        return x.transpose(1, 2).reshape(c['seqs'], c['kv'], span, c['dim'])
    q = s['q'].float().reshape(c['seqs'], c['kv'], -1, c['dim'])
    t = (q @ whole('k').transpose(-1, -2)) * c['dim'] ** -0.5
    behind = torch.arange(span, device='cuda') >= s['lengths'][:, None]
    t = t.masked_fill(behind[:, None, None], -math.inf)
    p = torch.exp(t - t.amax(-1, keepdim=True))
    v = whole('v').masked_fill(behind[:, None, :, None], 0.0)
    y = (p @ v) / p.sum(-1, keepdim=True)
    return {'y': y.reshape(c['seqs'], c['heads'], c['dim']).to(s['q'].dtype)}


def _packed_plain(s):
    c = s['case']
    group = c['heads'] // c['kv']
    y = torch.empty_like(s['q'])
    at = kt = 0
    for nq, nk in zip(s['new'], s['keys']):
        ahead = torch.ones((nq, nk), dtype=torch.bool, device='cuda').triu(nk - nq + 1) if c['causal'] else None
        for h in range(c['kv']):
            q = s['q'][at:at + nq, h * group:(h + 1) * group].float().transpose(0, 1)
            k, v = s['k'][kt:kt + nk, h].float(), s['v'][kt:kt + nk, h].float()
            t = (q.reshape(-1, c['dim']) @ k.t()).reshape(group, nq, nk) * c['dim'] ** -0.5
            if ahead is not None:
                t.masked_fill_(ahead, -math.inf)
            p = t.sub_(t.amax(-1, keepdim=True)).exp_()
            o = (p.reshape(-1, nk) @ v).reshape(group, nq, -1) / p.sum(-1, keepdim=True)
            y[at:at + nq, h * group:(h + 1) * group] = o.transpose(0, 1).to(y.dtype)
        at, kt = at + nq, kt + nk
    return {'y': y}


# --------------------------------------------------------------- the calls
_CALLS = []


def _package():
    if not _CALLS:
        path = str(Path(__file__).resolve().parents[1] / 'minimax-h3-2xt4_amd')
        if path not in sys.path:
            sys.path.insert(0, path)
        from w8a8 import kv_cache, packed_attention
        _CALLS.extend((kv_cache, packed_attention.packed_attention))
    return _CALLS


def _own(s):
    c = s['case']
    kv_cache, packed_attention = _package()
    if c['op'] == 'packed':
        return {'y': packed_attention(s['q'], s['k'], s['v'], s['starts'], s['k_starts'], causal=c['causal'])}
    cache = s['handle']
    if c['op'] == 'attend':
        return {'y': kv_cache.attend(s['q'], cache, s['table'], s['lengths'])}
    kv_cache.write(cache, s['k'], s['v'], s['table'], s['lengths'], s['starts'])
    if not c['read']:
        return {'k': cache.k, 'v': cache.v}
    k, v = kv_cache.read(cache, s['table'], s['k_starts'], sum(s['keys']), dtype=s['k'].dtype)
    return {'k': k, 'v': v}


def run(state):
    if own:
        return _own(state)
    return {'cache': _cache_plain, 'attend': _attend_plain, 'packed': _packed_plain}[state['case']['op']](state)


# ------------------------------------------------------------ exact values
def _exact_codes(x):
    """The value in 64 bits that a row's codes stand for; the stored scale is fp32."""
    x = x.double()
    ratio = float(torch.tensor(1.0, dtype=torch.float32) / 127)
    scale = (x.abs().max(-1, keepdim=True).values * ratio).float().clamp_min(1e-30).double()
    return torch.clamp(torch.round(x / scale), -128, 127) * scale


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c['op'] == 'packed':
        return {'y': _exact_packed(s)}
    cache = s['cache']

    def sequence(n, b):
        """[keys, kv, dim] of sequence b in 64 bits, as the cache holds it."""
        ids = s['table'][b, :-(-s['keys'][b] // c['page'])].long()
        x = cache[n].index_select(0, ids).double()
        if c['codes']:
            x *= cache[n + '_scale'].index_select(0, ids).double().unsqueeze(-1)
        return x.movedim(1, 2).flatten(0, 1)[:s['keys'][b]]

    if c['op'] == 'attend':
        out = torch.empty((c['seqs'], c['heads'], c['dim']), dtype=torch.float64, device='cuda')
        for b in range(c['seqs']):
            k, v = sequence('k', b), sequence('v', b)
            for h in range(c['heads']):
                j = h * c['kv'] // c['heads']
                w = torch.softmax(k[:, j] @ s['q'][b, h].double() / math.sqrt(c['dim']), 0)
                out[b, h] = w @ v[:, j]
        return {'y': out}
    new = [_exact_codes(s[n]) if c['codes'] else s[n].double() for n in ('k', 'v')]
    if c['read']:
        parts = ([], [])
        for b, count in enumerate(s['new']):
            first = int(s['starts'][b])
            for x, fresh, n in zip(parts, new, ('k', 'v')):
                x += [sequence(n, b)[:s['keys'][b] - count], fresh[first:first + count]]
        return {n: torch.cat(x) for n, x in zip(('k', 'v'), parts)}
    out = {n: cache[n].double() for n in ('k', 'v')}
    row = 0
    for b, count in enumerate(s['new']):
        ids = s['table'][b].tolist()
        position = s['keys'][b] - count
        while count:                          # a run of rows within one page
            run_ = min(count, c['page'] - position % c['page'])
            for fresh, n in zip(new, ('k', 'v')):
                at = position % c['page']
                out[n][ids[position // c['page']], :, at:at + run_] = fresh[row:row + run_].transpose(0, 1)
            row, position, count = row + run_, position + run_, count - run_
    return out


def _exact_packed(s):
    c = s['case']
    out = torch.empty(s['q'].shape, dtype=torch.float64, device='cuda')
    for b, (nq, nk) in enumerate(zip(s['new'], s['keys'])):
        q0, k0 = int(s['starts'][b]), int(s['k_starts'][b])
        block = max(1, min(nq, (1 << 26) // nk))
        for h in range(c['heads']):
            j = h * c['kv'] // c['heads']
            k, v = s['k'][k0:k0 + nk, j].double(), s['v'][k0:k0 + nk, j].double()
            for r in range(0, nq, block):
                n = min(block, nq - r)
                seen = nk - nq + r + n if c['causal'] else nk
                t = s['q'][q0 + r:q0 + r + n, h].double() @ k[:seen].t() / math.sqrt(c['dim'])
                if c['causal']:
                    last = torch.arange(nk - nq + r, nk - nq + r + n, device='cuda')
                    t[torch.arange(seen, device='cuda') > last[:, None]] = -math.inf
                out[q0 + r:q0 + r + n, h] = torch.softmax(t, 1) @ v[:seen]
    return out


# ------------------------------------------------------------ needed work
def work(case):
    c = case
    new, keys = _rows(c)
    rows, total = sum(new), sum(keys)
    if c['op'] == 'packed':
        pairs = sum(n * k - (n * (n - 1) // 2 if c['causal'] else 0) for n, k in zip(new, keys))
        return {'bytes': 2 * c['dim'] * (2 * rows * c['heads'] + 2 * total * c['kv']),
                'flops': 4 * pairs * c['heads'] * c['dim']}
    held = c['dim'] + 4 if c['codes'] else 2 * c['dim']        # bytes of one head's row in the cache
    if c['op'] == 'attend':
        return {'bytes': 2 * total * c['kv'] * held + 4 * c['seqs'] * c['heads'] * c['dim'],
                'flops': 4 * total * c['heads'] * c['dim']}
    per = 2 * rows * c['kv']
    out = {'bytes': per * (2 * c['dim'] + held), 'flops': per * c['dim'] * (3 if c['codes'] else 0)}
    if c['read']:
        out['bytes'] += 2 * total * c['kv'] * (held + 2 * c['dim'])
        out['flops'] += 2 * total * c['kv'] * c['dim'] if c['codes'] else 0
    return out
