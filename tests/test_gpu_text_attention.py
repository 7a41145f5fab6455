"""The cache and both attentions as a text encoder's serving step uses them:
prompts, their keys and values into pages, a prompt's next part behind its
cached keys, then tokens one by one. And the calls that are refused."""
import pytest
import torch

from attention_refs import attention64, bound, check, check_packed, starts_of, table_of
from w8a8 import _abi, axial_rope, kernels, kv_cache
from w8a8.kv_cache import KVCache
from w8a8.packed_attention import packed_attention

pytestmark = pytest.mark.gpu

HEADS, KV, DIM = 8, 2, 128


def projections(rows, dtype, seed):
    """Packed Q, K, V rows as one projection gives them."""
    g = torch.Generator().manual_seed(seed)
    return torch.randn((rows, HEADS + 2 * KV, DIM), generator=g).to(dtype).cuda()


@pytest.mark.parametrize('held,dtype', [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                        (torch.int8, torch.bfloat16), (torch.int8, torch.float16)])
def test_prompt_parts_and_tokens(gpu, held, dtype):
    """Every route gives the attention of the whole sequences: a prompt at once, its second part behind the
    cache's keys, and its last tokens one at a time. The reference runs over the keys and values that the
    cache holds (16 bits as they are, codes as their values), packed, in 64 bits."""
    total, part, tokens = [150, 40, 97], [60, 33, 1], 5
    st, starts = starts_of(total, 'cuda')
    rows = projections(st[-1], dtype, 3)
    inv, axis = axial_rope.ladder((DIM // 2,), device=gpu)
    pos = torch.cat([torch.arange(n) for n in total]).int()[:, None].cuda()
    q, k = axial_rope.rotate(rows[:, :HEADS], rows[:, HEADS:HEADS + KV], pos, inv, axis)
    v = rows[:, HEADS + KV:]
    table, pages = table_of(total, 16, torch.Generator().manual_seed(1), 'cuda')
    cache = KVCache.allocate(pages, 16, KV, DIM, dtype=held)

    def rows_of(first, last):
        """The packed rows [first[b], last[b]) of every sequence, and their starts."""
        ids = torch.cat([torch.arange(st[b] + f, st[b] + n) for b, (f, n) in enumerate(zip(first, last))]).cuda()
        return ids, starts_of([n - f for f, n in zip(first, last)], 'cuda')[1]

    def lengths(n):
        return torch.tensor(n, dtype=torch.int32, device='cuda')

    outs = torch.zeros_like(q)
    # the first part of every prompt, from the rows themselves; its keys go into pages
    ids, s = rows_of([0] * 3, part)
    outs[ids] = packed_attention(q[ids], k[ids], v[ids], s)
    kv_cache.write(cache, k[ids], v[ids], table, lengths(part), s)
    # the second part, up to the last tokens, over what the cache holds
    upto = [n - tokens for n in total]
    ids, s = rows_of(part, upto)
    kv_cache.write(cache, k[ids], v[ids], table, lengths(upto), s)
    ks, k_starts = starts_of(upto, 'cuda')
    ck, cv = kv_cache.read(cache, table, k_starts, ks[-1], dtype=dtype)
    outs[ids] = packed_attention(q[ids], ck, cv, s, k_starts)
    # the last tokens, one by one
    for i in range(tokens):
        n = [m + i + 1 for m in upto]
        ids, _ = rows_of([m - 1 for m in n], n)
        kv_cache.write(cache, k[ids], v[ids], table, lengths(n))
        outs[ids] = kv_cache.attend(q[ids], cache, table, lengths(n))
    hk, hv = kv_cache.read(cache, table, starts, st[-1], dtype=dtype)
    if held != torch.int8:
        assert torch.equal(hk, k) and torch.equal(hv, v)
        check_packed(outs, q, hk, hv, st, st, True, DIM ** -0.5)
        return
    # with codes the first parts saw the rows themselves, the second what `read` rounds to 16 bits
    for b in range(3):
        a, z = st[b] + part[b], st[b + 1] - tokens
        check_packed(outs[st[b]:a], q[st[b]:a], k[st[b]:a], v[st[b]:a], [0, part[b]], [0, part[b]], True, DIM ** -0.5)
        check_packed(outs[a:z], q[a:z], hk[st[b]:z], hv[st[b]:z], [0, z - a], [0, z - st[b]], True, DIM ** -0.5)
    for b in range(3):   # the tokens see the codes' exact values
        ids = torch.arange(total[b], device='cuda')
        at, off = table[b].long()[ids // 16], ids % 16
        for h in range(HEADS):
            j = h // (HEADS // KV)
            vs = cache.v_scale[at, j, off].double()[:, None]
            k64, v64 = cache.k[at, j, off].double() * cache.k_scale[at, j, off].double()[:, None], cache.v[at, j, off].double()
            first = torch.arange(total[b] - tokens + 1, total[b] + 1, device='cuda')
            z = slice(st[b + 1] - tokens, st[b + 1])
            o, parts = attention64(q[z, h].double(), k64, v64 * vs, DIM ** -0.5, first, codes_scale=v64.abs() * vs.max())
            check(outs[z, h], o, bound(o, parts, dtype), f'tokens of sequence {b} head {h}')


def test_refusals(gpu):
    cache = KVCache.allocate(3, 16, 2, 64)
    codes = KVCache.allocate(3, 16, 2, 64, dtype=torch.int8)
    table = torch.zeros((2, 2), dtype=torch.int32, device='cuda')
    n, starts = (torch.tensor(x, dtype=torch.int32, device='cuda') for x in ([1, 2], [0, 1, 3]))
    x, q = torch.zeros((3, 2, 64), device='cuda').half(), torch.zeros((2, 4, 64), device='cuda').half()
    bad = [
        lambda: kv_cache.write(cache, x.bfloat16(), x.bfloat16(), table, n, starts),
        lambda: kv_cache.write(codes, x.float(), x.float(), table, n, starts),
        lambda: kv_cache.write(cache, x, x[:2], table, n, starts),
        lambda: kv_cache.write(codes, x, x.bfloat16(), table, n, starts),
        lambda: kv_cache.write(cache, x[:, :1], x[:, :1], table, n, starts),
        lambda: kv_cache.write(cache, x[..., :32], x[..., :32], table, n, starts),
        lambda: kv_cache.write(cache, x, x, table, n),
        lambda: kv_cache.write(cache, x, x, table.long(), n, starts),
        lambda: kv_cache.write(cache, x, x, table[0], n, starts),
        lambda: kv_cache.write(cache, x, x, table, n.long(), starts),
        lambda: kv_cache.write(cache, x, x, table, n[:1], starts),
        lambda: kv_cache.write(cache, x, x, table, n, starts[:2]),
        lambda: kv_cache.write(cache, x, x, table, n, starts.long()),
        lambda: kv_cache.write(cache, x, x, table, n.cpu(), starts),
        lambda: kv_cache.read(cache, table, starts, 3, dtype=torch.bfloat16),
        lambda: kv_cache.read(codes, table, starts, 3, dtype=torch.float32),
        lambda: kv_cache.read(cache, table, starts[:2], 3),
        lambda: kv_cache.read(cache, table, starts, 3, out=(x, x[:2])),
        lambda: kv_cache.read(cache, table, starts, 3, out=(x, x.bfloat16())),
        lambda: kv_cache.read(cache, table, starts, 3, out=(x.transpose(1, 2).contiguous().transpose(1, 2), x)),
        lambda: kv_cache.read(cache, table, starts, 3, out=(x[:1].expand(3, 2, 64), x)),
        lambda: kv_cache.attend(q[:1], cache, table, n),
        lambda: kv_cache.attend(q[:, :3], cache, table, n),
        lambda: kv_cache.attend(q[:, :0], cache, table, n),
        lambda: kv_cache.attend(q[..., :32], cache, table, n),
        lambda: kv_cache.attend(q.bfloat16(), cache, table, n),
        lambda: kv_cache.attend(q.float(), codes, table, n),
        lambda: kv_cache.attend(q, cache, table, n.float()),
        lambda: kv_cache.attend(q, cache, table, n, scale=0.0),
        lambda: kv_cache.attend(q, cache, table, n, scale=-0.1),
        lambda: kv_cache.attend(q, cache, table, n, scale=float('nan')),
        lambda: kv_cache.attend(q, cache, table, n, out=q[:1]),
        lambda: kv_cache.attend(q, cache, table, n, out=q.bfloat16()),
        lambda: kv_cache.attend(q, cache, table, n, out=torch.empty((2, 64, 4), device='cuda').half().transpose(1, 2)),
        lambda: packed_attention(q, x, x, starts),
        lambda: packed_attention(x, x, x.bfloat16(), starts),
        lambda: packed_attention(x.float(), x.float(), x.float(), starts),
        lambda: packed_attention(x, x, x[:2], starts, starts),
        lambda: packed_attention(x, x[..., :32], x[..., :32], starts),
        lambda: packed_attention(x[..., :60], x[..., :60], x[..., :60], starts),
        lambda: packed_attention(x[:, :1], x, x, starts),
        lambda: packed_attention(x[:, :0], x, x, starts),
        lambda: packed_attention(x, x, x, starts.long()),
        lambda: packed_attention(x, x, x, starts, starts[:2]),
        lambda: packed_attention(x, x, x, starts[:0]),
        lambda: packed_attention(x, x, x, starts, scale=float('inf')),
        lambda: packed_attention(x, x, x, starts, out=x[:2]),
        lambda: packed_attention(x, x, x, starts, out=x[:1].expand(3, 2, 64)),
        lambda: packed_attention(x[0], x, x, starts),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print(i)   # (the call that was taken)


def test_writes_are_counted(gpu):
    """Autograd sees that a tensor it saved has changed."""
    cache = KVCache.allocate(3, 16, 2, 64, dtype=torch.int8)
    table = torch.zeros((1, 2), dtype=torch.int32, device='cuda')
    n, starts = (torch.tensor(t, dtype=torch.int32, device='cuda') for t in ([3], [0, 3]))
    x, q = torch.zeros((3, 2, 64), device='cuda').half(), torch.zeros((1, 4, 64), device='cuda').half()
    before = [t._version for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    kv_cache.write(cache, x, x, table, n, starts)
    assert all(t._version > b for t, b in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), before))
    outs = [torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(q), torch.zeros_like(x)]
    before = [t._version for t in outs]
    kv_cache.read(cache, table, starts, 3, out=(outs[0], outs[1]))
    kv_cache.attend(q, cache, table, n, out=outs[2])
    packed_attention(x, x, x, starts, out=outs[3])
    assert all(t._version > b for t, b in zip(outs, before))


def test_host_routes_give_the_same_bits(gpu):
    """The native calls and the Python route that they fall back to."""
    g = torch.Generator().manual_seed(2)
    total = [40, 0, 90]
    st, starts = starts_of(total, 'cuda')
    table, pages = table_of(total, 16, g, 'cuda')
    n = torch.tensor(total, dtype=torch.int32, device='cuda')
    for held, dtype in ((torch.float16,) * 2, (torch.int8, torch.bfloat16)):
        rows = projections(st[-1], dtype, 4)
        q, k, v = rows[:, :HEADS], rows[:, HEADS:HEADS + KV], rows[:, HEADS + KV:]
        one, two = (KVCache.allocate(pages, 16, KV, DIM, dtype=held) for _ in range(2))
        args = (one.k, one.v, one.k_scale, one.v_scale)
        native = _abi.native()
        assert native.cache_write(*args, k, v, table, n, starts) is True
        kernels.cache_write(two, k, v, table, n, starts)
        assert all(a is None or torch.equal(a, b) for a, b in zip(args, (two.k, two.v, two.k_scale, two.v_scale)))
        for a, b in zip(native.cache_read(*args, table, starts, st[-1], dtype),
                        kernels.cache_read(two, table, starts, st[-1], dtype=dtype)):
            assert torch.equal(a, b)
        x = rows[:3, :HEADS]
        out = torch.empty_like(x)
        for scale in (None, 0.2):
            want = kernels.cache_attend(x, two, table, n, scale=scale)
            assert torch.equal(native.cache_attend(*args, x, table, n, scale, None), want)
            assert native.cache_attend(*args, x, table, n, scale, out) is out and torch.equal(out, want)
            want = kernels.packed_attention(q, k, v, starts, causal=False, scale=scale)
            assert torch.equal(native.packed_attention(q, k, v, starts, starts, False, scale, None), want)


def test_outputs_between_the_inputs(gpu):
    """Outputs may be columns of the buffer whose other columns are read or written."""
    total = [33, 70]
    st, starts = starts_of(total, 'cuda')
    table, pages = table_of(total, 16, torch.Generator().manual_seed(8), 'cuda')
    n = torch.tensor(total, dtype=torch.int32, device='cuda')
    rows = torch.cat([projections(st[-1], torch.bfloat16, 5), torch.zeros((st[-1], HEADS, DIM)).bfloat16().cuda()], 1)
    q, k, v = rows[:, :HEADS], rows[:, HEADS:HEADS + KV], rows[:, HEADS + KV:HEADS + 2 * KV]
    out = rows[:, HEADS + 2 * KV:]
    want = packed_attention(q.clone(), k.clone(), v.clone(), starts)
    packed_attention(q, k, v, starts, out=out)
    assert torch.equal(out, want)
    with pytest.raises(RuntimeError, match='overlaps an input'):
        packed_attention(q, k, v, starts, out=rows[:, 1:HEADS + 1])
    cache = KVCache.allocate(pages, 16, KV, DIM, dtype=torch.int8)
    kv_cache.write(cache, k, v, table, n, starts)
    both = torch.zeros((st[-1], 2 * KV, DIM), dtype=torch.bfloat16, device='cuda')
    kv_cache.read(cache, table, starts, st[-1], out=(both[:, :KV], both[:, KV:]))
    for got, x in zip((both[:, :KV], both[:, KV:]), kv_cache.read(cache, table, starts, st[-1], dtype=torch.bfloat16)):
        assert torch.equal(got, x)
    with pytest.raises(RuntimeError, match='overlap'):
        kv_cache.read(cache, table, starts, st[-1], out=(both[:, :KV], both[:, KV - 1:2 * KV - 1]))
    buf = torch.zeros((2, 2 * HEADS, DIM), dtype=torch.bfloat16, device='cuda')
    buf[:, :HEADS] = q[:2]
    kv_cache.attend(buf[:, :HEADS], cache, table, n, out=buf[:, HEADS:])
    assert torch.equal(buf[:, HEADS:], kv_cache.attend(q[:2], cache, table, n))


@pytest.mark.parametrize('held,dtype', [(torch.float16, torch.float16), (torch.int8, torch.bfloat16)])
def test_calls_at_once(gpu, held, dtype):
    """Two streams whose calls share keys between workgroups, each with workspaces of its own: the bits of
    calls one after the other."""
    def setup(seed, total):
        rows = projections(sum(total), dtype, seed)
        st, starts = starts_of(total, 'cuda')
        table, pages = table_of(total, 32, torch.Generator().manual_seed(seed), 'cuda')
        cache = KVCache.allocate(pages, 32, KV, DIM, dtype=held)
        lengths = torch.tensor(total, dtype=torch.int32, device='cuda')
        few = [min(n, 20) for n in total]
        return dict(k=rows[:, HEADS:HEADS + KV], v=rows[:, HEADS + KV:], q=rows[:sum(few), :HEADS], cache=cache,
                    table=table, lengths=lengths, starts=starts, rows=sum(total), few=starts_of(few, 'cuda')[1])

    def run(s):
        kv_cache.write(s['cache'], s['k'], s['v'], s['table'], s['lengths'], s['starts'])
        k, v = kv_cache.read(s['cache'], s['table'], s['starts'], s['rows'], dtype=dtype)
        n = s['lengths'].shape[0]
        return k, v, packed_attention(s['q'], k, v, s['few'], s['starts']), \
            kv_cache.attend(s['q'][:n], s['cache'], s['table'], s['lengths'])

    sets = [setup(1, [3000, 17, 1200]), setup(2, [5000, 900])]
    for s in sets:
        lib = _abi.load()
        assert lib.w8a8_packed_attention_workspace_size(s['q'].shape[0], s['rows'], s['few'].numel() - 1, HEADS, KV, DIM) > 0
        assert lib.w8a8_cache_attend_workspace_size(s['lengths'].numel(), HEADS, KV, DIM, s['table'].shape[1] * 32) > 0
    want = [run(s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(run(s))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(outs, want[i % 2])), i
