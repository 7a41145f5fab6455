"""The paged key-value cache: writing, reading back, and one token's attention
over it, against 64 bits (tolerances: attention_refs)."""
import math

import pytest
import torch

from attention_refs import attention64, bound, check, quantize64, starts_of, table_of
from w8a8 import kv_cache
from w8a8.kv_cache import KVCache

pytestmark = pytest.mark.gpu

HELD = [torch.float16, torch.bfloat16, torch.int8]


def kv_rows(dtype, rows, heads, dim, seed=0):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn((rows, heads, dim), generator=g) * (10.0 ** torch.randint(-3, 2, (rows, heads, 1), generator=g))
    v = torch.randn((rows, heads, dim), generator=g)
    return k.to(dtype).cuda(), v.to(dtype).cuda()


def put(cache, k, v, table, page, first, rows):
    """The plain write of rows into keys first, first + 1, ... of a sequence with this table row."""
    for i in range(rows):
        j = first + i
        at, off = int(table[j // page]), j % page
        for name, x in (('k', k[i]), ('v', v[i])):
            if cache.codes:
                getattr(cache, name)[at, :, off], getattr(cache, name + '_scale')[at, :, off] = quantize64(x)
            else:
                getattr(cache, name)[at, :, off] = x


def same(a, b):
    for n in ('k', 'v', 'k_scale', 'v_scale'):
        x, y = getattr(a, n), getattr(b, n)
        assert (x is None) == (y is None)
        assert x is None or torch.equal(x, y), n


def twin(pages, page, heads, dim, held):
    return tuple(KVCache.allocate(pages, page, heads, dim, dtype=held) for _ in range(2))


@pytest.mark.parametrize('held', HELD)
@pytest.mark.parametrize('page,heads,dim', [(16, 8, 128), (48, 3, 72), (64, 1, 64), (32, 28, 80), (16, 5, 256), (128, 2, 8),
                                            (16, 9, 136)])
def test_write_and_read(gpu, held, page, heads, dim):
    dtype = torch.bfloat16 if held == torch.int8 else held
    new, before = [20, 0, 1, 37], [5, 3, 64, 0]
    total = [a + b for a, b in zip(new, before)]
    table, pages = table_of(total, page, torch.Generator().manual_seed(dim), 'cuda')
    cache, want = twin(pages, page, heads, dim, held)
    st, starts = starts_of(new, 'cuda')
    k, v = kv_rows(dtype, st[-1] + 5, heads, dim, seed=page)   # five rows behind the last sequence
    lengths = torch.tensor(total, dtype=torch.int32, device='cuda')
    kv_cache.write(cache, k, v, table, lengths, starts)
    for b, n in enumerate(new):
        put(want, k[st[b]:], v[st[b]:], table[b].tolist(), page, before[b], n)
    same(cache, want)
    # and back: whole sequences, the untouched keys being zeros
    ks, k_starts = starts_of(total, 'cuda')
    rk, rv = kv_cache.read(cache, table, k_starts, ks[-1] + 3, dtype=dtype)
    for b, n in enumerate(total):
        for i in range(n):
            at, off = int(table[b, i // page]), i % page
            for got, name in ((rk, 'k'), (rv, 'v')):
                x = getattr(cache, name)[at, :, off]
                if cache.codes:
                    x = (x.float() * getattr(cache, name + '_scale')[at, :, off][:, None]).to(dtype)
                assert torch.equal(got[ks[b] + i], x), (b, i, name)
    assert not bool(rk[ks[-1]:].any()) and not bool(rv[ks[-1]:].any())
    out = tuple(torch.full_like(rk, 3.0) for _ in range(2))
    kv_cache.read(cache, table, k_starts, ks[-1] + 3, out=out)
    assert torch.equal(out[0][:ks[-1]], rk[:ks[-1]]) and bool((out[1][ks[-1]:] == 3.0).all())


@pytest.mark.parametrize('held', HELD)
def test_one_row_a_sequence(gpu, held):
    dtype = torch.float16 if held == torch.int8 else held
    total = [1, 16, 17, 40, 33]
    table, pages = table_of(total, 16, torch.Generator().manual_seed(1), 'cuda')
    cache, want = twin(pages, 16, 8, 128, held)
    k, v = kv_rows(dtype, 5, 8, 128)
    kv_cache.write(cache, k, v, table, torch.tensor(total, dtype=torch.int32, device='cuda'))
    for b, n in enumerate(total):
        put(want, k[b:], v[b:], table[b].tolist(), 16, n - 1, 1)
    same(cache, want)


@pytest.mark.parametrize('sequences', [63, 64, 65, 130, 5000])
def test_many_sequences(gpu, sequences):
    """Empty ones among them, and rows behind the last."""
    g = torch.Generator().manual_seed(sequences)
    new = torch.randint(0, 6, (sequences,), generator=g)
    new[0] = new[sequences // 2] = new[-1] = 0
    before = torch.randint(0, 20, (sequences,), generator=g)
    total = new + before
    table, pages = table_of(total.tolist(), 16, g, 'cuda')
    cache, want = twin(pages, 16, 2, 64, torch.float16)
    st, starts = starts_of(new.tolist(), 'cuda')
    k, v = kv_rows(torch.float16, st[-1] + 70, 2, 64, seed=sequences)
    kv_cache.write(cache, k, v, table, total.int().cuda(), starts)
    b = torch.repeat_interleave(torch.arange(sequences), new)
    key = (before[b] + torch.arange(st[-1]) - torch.tensor(st)[b]).cuda()
    page = table[b.cuda(), key // 16].long()
    want.k[page, :, key % 16], want.v[page, :, key % 16] = k[:st[-1]], v[:st[-1]]
    same(cache, want)
    ks, k_starts = starts_of(total.tolist(), 'cuda')
    rk, rv = kv_cache.read(cache, table, k_starts, ks[-1] + 70)
    b = torch.repeat_interleave(torch.arange(sequences), total)
    key = (torch.arange(ks[-1]) - torch.tensor(ks)[b]).cuda()
    page = table[b.cuda(), key // 16].long()
    assert torch.equal(rk[:ks[-1]], cache.k[page, :, key % 16]) and torch.equal(rv[:ks[-1]], cache.v[page, :, key % 16])
    assert not bool(rk[ks[-1]:].any()) and not bool(rv[ks[-1]:].any())


@pytest.mark.parametrize('single', [False, True])
@pytest.mark.parametrize('held,heads,dim', [(torch.float16, 1, 128), (torch.int8, 1, 72), (torch.int8, 5, 64),
                                            (torch.bfloat16, 3, 40), (torch.int8, 2, 128), (torch.int8, 1, 256)])
def test_many_rows_of_few_heads(gpu, held, heads, dim, single):
    """A wave has several rows: of a sequence or of many, empty ones and absent pages among them."""
    dtype = torch.bfloat16 if held == torch.int8 else held
    g = torch.Generator().manual_seed(dim)
    new = torch.ones(4500, dtype=torch.int64) if single else torch.cat(
        [torch.randint(0, 4, (200,), generator=g), torch.tensor([4000, 0, 0, 33]), torch.randint(0, 40, (70,), generator=g)])
    n = len(new)
    before = torch.randint(0, 40, (n,), generator=g)
    total = new + before
    table, pages = table_of(total.tolist(), 32, g, 'cuda')
    table[::7, 0] = -1
    cache, want = twin(pages, 32, heads, dim, held)
    st, starts = starts_of(new.tolist(), 'cuda')
    k, v = kv_rows(dtype, st[-1] if single else st[-1] + 77, heads, dim, seed=dim)
    kv_cache.write(cache, k, v, table, total.int().cuda(), None if single else starts)
    b = torch.repeat_interleave(torch.arange(n), new)
    key = (before[b] + torch.arange(st[-1]) - torch.tensor(st)[b]).cuda()
    page = table[b.cuda(), key // 32].long()
    there, at, off = page >= 0, page[page >= 0], key[page >= 0] % 32
    for name, x in (('k', k), ('v', v)):
        x = x[:st[-1]][there]
        if cache.codes:
            getattr(want, name)[at, :, off], getattr(want, name + '_scale')[at, :, off] = quantize64(x)
        else:
            getattr(want, name)[at, :, off] = x
    same(cache, want)
    ks, k_starts = starts_of(total.tolist(), 'cuda')
    rk, rv = kv_cache.read(cache, table, k_starts, ks[-1] + 77, dtype=dtype)
    b = torch.repeat_interleave(torch.arange(n), total)
    key = (torch.arange(ks[-1]) - torch.tensor(ks)[b]).cuda()
    page = table[b.cuda(), key // 32].long()
    for got, name in ((rk, 'k'), (rv, 'v')):
        x = getattr(cache, name)[page.clamp_min(0), :, key % 32]
        if cache.codes:
            x = (x.float() * getattr(cache, name + '_scale')[page.clamp_min(0), :, key % 32][..., None]).to(dtype)
        assert torch.equal(got[:ks[-1]], torch.where((page >= 0)[:, None, None], x, torch.zeros_like(x))), name
        assert not bool(got[ks[-1]:].any())
    out = tuple(torch.full_like(rk, 3.0) for _ in range(2))
    kv_cache.read(cache, table, k_starts, ks[-1] + 77, out=out)
    assert all(torch.equal(o[:ks[-1]], r[:ks[-1]]) and bool((o[ks[-1]:] == 3.0).all()) for o, r in zip(out, (rk, rv)))


def test_places_that_are_not_there(gpu):
    """Keys outside of the table, absent pages and pages outside of the cache are not written."""
    cache, want = twin(4, 16, 2, 64, torch.float16)
    table = torch.tensor([[2, -1], [4, 1], [1000000, 0]], dtype=torch.int32, device='cuda')
    k, v = kv_rows(torch.float16, 60, 2, 64)
    _, starts = starts_of([20, 20, 20], 'cuda')
    lengths = torch.tensor([20, 20, 40], dtype=torch.int32, device='cuda')
    kv_cache.write(cache, k, v, table, lengths, starts)
    put(want, k, v, [2], 16, 0, 16)
    put(want, k[36:], v[36:], [-1, 1], 16, 16, 4)
    put(want, k[40:], v[40:], [-1, 0], 16, 20, 12)   # the last 8 lie behind the table
    same(cache, want)
    lengths = torch.tensor([10, -5, 0], dtype=torch.int32, device='cuda')   # more new rows than keys
    kv_cache.write(cache, k, v, table, lengths, starts)
    put(want, k[10:], v[10:], [2], 16, 0, 10)
    same(cache, want)
    rk, rv = kv_cache.read(cache, table, torch.tensor([0, 40, 60, 60], dtype=torch.int32, device='cuda'), 60)
    assert torch.equal(rk[:16], cache.k[2].transpose(0, 1)) and not bool(rk[16:40].any())
    assert not bool(rk[40:56].any()) and torch.equal(rv[56:60], cache.v[1, :, :4].transpose(0, 1))


@pytest.mark.parametrize('heads', [1, 8])
def test_starts_and_lengths_out_of_range_stay_in_bounds(gpu, heads):
    """Whatever starts and lengths hold, only the cache's pages and the rows are touched."""
    big = torch.full((2, 12, heads, 16, 64), 7.0, dtype=torch.float16, device='cuda')
    cache = KVCache(big[0, 4:8], big[1, 4:8])
    rows = torch.full((2, 7000, heads, 64), 7.0, dtype=torch.float16, device='cuda')
    k, v = rows[0, 1000:6000], rows[1, 1000:6000]
    low, high = -2 ** 31, 2 ** 31 - 1
    table = torch.tensor([[0, 3], [1, 4], [high, 2], [low, -1]], dtype=torch.int32, device='cuda')
    for starts in ([0, 9000, 9000, 9000, 9000], [0, -5, 3, 2, 4900], [high, low, 0, high, low], [5, 4, 3, 2, 1],
                   [low, high, high, high, high], [0, 10, 20, 30, 40]):
        for lengths in ([20, 40, 30, 5], [high] * 4, [low] * 4, [0, -1, 33, 1000]):
            s, n = (torch.tensor(t, dtype=torch.int32, device='cuda') for t in (starts, lengths))
            kv_cache.write(cache, torch.zeros_like(k), torch.zeros_like(v), table, n, s)
            kv_cache.read(cache, table, s, 5000, out=(k, v))
            kv_cache.attend(torch.zeros((4, heads, 64), dtype=torch.float16, device='cuda'), cache, table, n)
    assert bool((big[:, :4] == 7.0).all()) and bool((big[:, 8:] == 7.0).all())
    assert bool((rows[:, :1000] == 7.0).all()) and bool((rows[:, 6000:] == 7.0).all())


def test_rows_that_are_not_finite(gpu):
    cache, _ = twin(1, 16, 2, 64, torch.int8)
    k, v = kv_rows(torch.bfloat16, 4, 2, 64)
    k[1, 0, 5], v[2, 1, 63], v[3] = math.inf, math.nan, 0.0
    table = torch.zeros((1, 1), dtype=torch.int32, device='cuda')
    lengths, starts = (torch.tensor(x, dtype=torch.int32, device='cuda') for x in ([4], [0, 4]))
    kv_cache.write(cache, k, v, table, lengths, starts)
    rk, rv = kv_cache.read(cache, table, starts, 4, dtype=torch.bfloat16)
    assert bool(torch.isnan(rk[1, 0]).all()) and bool(torch.isfinite(rk[1, 1]).all())
    assert bool(torch.isnan(rv[2, 1]).all()) and not bool(rv[3].any())
    assert float(cache.v_scale[0, 0, 3]) == pytest.approx(1e-30)


def views(held, pages, page, heads, dim):
    """A cache whose keys and values, and scales, share buffers, tokens before heads."""
    buf = torch.zeros((pages, page, 2, heads, dim), dtype=held, device='cuda').permute(2, 0, 3, 1, 4)
    if held != torch.int8:
        return KVCache(buf[0], buf[1])
    sc = torch.zeros((pages, 2, heads, page), dtype=torch.float32, device='cuda')
    return KVCache(buf[0], buf[1], sc[:, 0], sc[:, 1])


# ------------------------------------------------------------ attention
def filled(held, pages, page, heads, dim, dtype, seed=0):
    cache = KVCache.allocate(pages, page, heads, dim, dtype=held)
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((pages, heads, page, dim), generator=g).to(dtype).cuda() for _ in range(2))
    v *= (10.0 ** torch.randint(-2, 2, (pages, heads, page, 1), generator=g)).to(dtype).cuda()
    if held == torch.int8:
        for name, x in (('k', k), ('v', v)):
            c, s = quantize64(x)
            getattr(cache, name).copy_(c)
            getattr(cache, name + '_scale').copy_(s)
    else:
        cache.k.copy_(k)
        cache.v.copy_(v)
    return cache


def check_attend(y, q, cache, table, lengths, scale, what=''):
    page, group = cache.page_size, q.shape[1] // cache.heads
    for b, n in enumerate(lengths):
        n = min(max(n, 0), table.shape[1] * page)
        ids = [(int(table[b, j // page]), j % page) for j in range(n)]
        ids = [(p, o) for p, o in ids if 0 <= p < cache.k.shape[0]]
        pg = torch.tensor([p for p, _ in ids], dtype=torch.long, device='cuda')
        of = torch.tensor([o for _, o in ids], dtype=torch.long, device='cuda')
        for h in range(cache.heads):
            k, v = cache.k[pg, h, of].double(), cache.v[pg, h, of].double()
            lost = None
            if cache.codes:
                k, vs = k * cache.k_scale[pg, h, of].double()[:, None], cache.v_scale[pg, h, of].double()[:, None]
                lost = v.abs() * (vs.max() if len(ids) else 0.0)
                v = v * vs
            for i in range(group):
                o, parts = attention64(q[b, h * group + i][None].double(), k, v, scale, codes_scale=lost)
                check(y[b, h * group + i][None], o, bound(o, parts, q.dtype), f'{what} sequence {b} head {h * group + i}')


def attend_case(held, dtype, page, heads, kv, dim, lengths, seed=0):
    table, pages = table_of(lengths, page, torch.Generator().manual_seed(seed), 'cuda')
    cache = filled(held, pages, page, kv, dim, dtype, seed)
    q = (torch.randn((len(lengths), heads, dim), generator=torch.Generator().manual_seed(seed + 1)) * 1.5).to(dtype).cuda()
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    y = kv_cache.attend(q, cache, table, n)
    check_attend(y, q, cache, table, lengths, dim ** -0.5)
    assert torch.equal(kv_cache.attend(q, cache, table, n), y)   # the same bits every time
    return q, cache, table, n, y


TYPES = [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.int8, torch.float16),
         (torch.int8, torch.bfloat16)]


@pytest.mark.parametrize('held,dtype', TYPES)
@pytest.mark.parametrize('dim', [8, 24, 64, 72, 80, 96, 128, 136, 256])
def test_attend_dims(gpu, held, dtype, dim):
    attend_case(held, dtype, 16, 4, 2, dim, [70, 1, 33, 130], seed=dim)


@pytest.mark.parametrize('held,dtype', TYPES)
@pytest.mark.parametrize('page', [16, 48, 64, 256])
@pytest.mark.parametrize('lengths', [[1], [0], [15, 16, 17], [0, 5, 0, 128, 129, 0], [354], [1000, 3, 127]])
def test_attend_lengths(gpu, held, dtype, page, lengths):
    attend_case(held, dtype, page, 8, 1, 128, lengths, seed=page)


@pytest.mark.parametrize('heads,kv', [(1, 1), (7, 7), (16, 1), (17, 1), (40, 2), (64, 8)])
def test_attend_groups(gpu, heads, kv):
    attend_case(torch.float16, torch.float16, 32, heads, kv, 64, [100, 40])
    attend_case(torch.int8, torch.bfloat16, 32, heads, kv, 64, [100, 40])


@pytest.mark.parametrize('held,dtype', TYPES)
def test_attend_many_sequences(gpu, held, dtype):
    attend_case(held, dtype, 16, 2, 1, 64, [(37 * i) % 90 for i in range(150)])


@pytest.mark.parametrize('held,dtype', TYPES)
def test_attend_shared_by_workgroups(gpu, held, dtype):
    """Long sequences beside short ones: several workgroups join their sums."""
    attend_case(held, dtype, 64, 8, 2, 128, [20000, 5, 0, 9001])


def test_attend_layouts(gpu):
    table, pages = table_of([50, 90], 16, torch.Generator().manual_seed(2), 'cuda')
    n = torch.tensor([50, 90], dtype=torch.int32, device='cuda')
    for held, dtype in TYPES:
        cache = filled(held, pages, 16, 2, 64, dtype)
        q = torch.randn((2, 4, 64), generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
        want = kv_cache.attend(q, cache, table, n)
        other = views(held, pages, 16, 2, 64)
        for name in ('k', 'v', 'k_scale', 'v_scale'):
            if getattr(cache, name) is not None:
                getattr(other, name).copy_(getattr(cache, name))
        assert torch.equal(kv_cache.attend(q, other, table, n), want)
        buf = torch.zeros((2, 6, 64), dtype=dtype, device='cuda')
        out = buf[:, 1:5]
        kv_cache.attend(q.transpose(0, 1).contiguous().transpose(0, 1), cache, table, n, out=out)
        assert torch.equal(out, want) and not bool(buf[:, 0].any()) and not bool(buf[:, 5].any())
        wide = torch.full((4, table.shape[1] + 9), -1, dtype=torch.int32, device='cuda')
        wide[::2, :table.shape[1]] = table
        assert torch.equal(kv_cache.attend(q, cache, wide[::2], n), want)
        k, v = kv_rows(dtype, 2, 2, 64)
        kv_cache.write(cache, k, v, table, n)
        kv_cache.write(other, k, v, table, n)
        same(KVCache(other.k.contiguous(), other.v.contiguous(), *(t.contiguous() for t in (other.k_scale, other.v_scale)
                                                                   if t is not None)), cache)


def test_attend_garbage_behind_the_end(gpu):
    """What lies behind a sequence's end or in no page has no effect."""
    for held, dtype in TYPES:
        table, pages = table_of([33, 100], 16, torch.Generator().manual_seed(4), 'cuda', width=10)
        cache = filled(held, pages, 16, 2, 64, dtype)
        q = torch.randn((2, 4, 64), generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
        n = torch.tensor([33, 100], dtype=torch.int32, device='cuda')
        want = kv_cache.attend(q, cache, table, n)
        used = {(int(table[b, j // 16]), j % 16) for b, m in ((0, 33), (1, 100)) for j in range(m)}
        for p in range(pages):
            for o in range(16):
                if (p, o) in used:
                    continue
                if cache.codes:
                    cache.k_scale[p, :, o] = cache.v_scale[p, :, o] = math.nan
                else:
                    cache.k[p, :, o], cache.v[p, :, o] = math.nan, math.inf
        assert torch.equal(kv_cache.attend(q, cache, table, n), want)
        # an absent page in the middle, pages outside of the cache, lengths behind the table
        table[1, 2], table[1, 4] = -1, pages
        n = torch.tensor([33, 100], dtype=torch.int32, device='cuda')
        check_attend(kv_cache.attend(q, cache, table, n), q, cache, table, [33, 100], 0.125)
        narrow = table[:, :2].contiguous()
        n = torch.tensor([1000000, -3], dtype=torch.int32, device='cuda')
        y = kv_cache.attend(q, cache, narrow, n)
        check_attend(y, q, cache, narrow, [32, 0], 0.125)
        assert not bool(y[1].any())
        none = kv_cache.attend(q, cache, table[:, :0], n)
        assert not bool(none.any())


def test_attend_visible_nan(gpu):
    for held, dtype in TYPES:
        table, pages = table_of([40], 16, torch.Generator().manual_seed(4), 'cuda')
        cache = filled(held, pages, 16, 2, 64, dtype)
        page = int(table[0, 1])
        if cache.codes:
            cache.v_scale[page, 0, 3] = math.nan
        else:
            cache.v[page, 0, 3] = math.nan
        q = torch.randn((1, 4, 64), generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
        y = kv_cache.attend(q, cache, table, torch.tensor([40], dtype=torch.int32, device='cuda'))
        assert bool(torch.isnan(y[0, :2]).all()) and bool(torch.isfinite(y[0, 2:]).all())


@pytest.mark.parametrize('held,dtype', TYPES)
def test_attend_values_of_any_size(gpu, held, dtype):
    """Codes keep their precision whatever the values' size, and the other way round."""
    for size in (1e-6, 1e3) if dtype == torch.float16 else (1e-30, 1e30):
        table, pages = table_of([100], 16, torch.Generator().manual_seed(4), 'cuda')
        cache = filled(held, pages, 16, 1, 64, dtype)
        (cache.v_scale if cache.codes else cache.v).mul_(size)
        q = torch.randn((1, 4, 64), generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
        n = torch.tensor([100], dtype=torch.int32, device='cuda')
        check_attend(kv_cache.attend(q, cache, table, n), q, cache, table, [100], 0.125)


def test_far_pages(gpu):
    """Pages whose offsets pass 32 bits."""
    cache = KVCache.allocate(300000, 16, 8, 128, dtype=torch.int8)   # 4.9 GB each
    table = torch.tensor([[299999, 5, 270000]], dtype=torch.int32, device='cuda')
    k, v = kv_rows(torch.float16, 40, 8, 128)
    n, starts = (torch.tensor(x, dtype=torch.int32, device='cuda') for x in ([40], [0, 40]))
    kv_cache.write(cache, k, v, table, n, starts)
    rk, _ = kv_cache.read(cache, table, starts, 40)
    c, s = quantize64(k)
    assert torch.equal(rk, (c.float() * s[..., None]).half())
    q = torch.randn((1, 16, 128), generator=torch.Generator().manual_seed(3)).half().cuda()
    y = kv_cache.attend(q, cache, table, n)
    small = KVCache.allocate(3, 16, 8, 128, dtype=torch.int8)
    near = torch.tensor([[0, 1, 2]], dtype=torch.int32, device='cuda')
    kv_cache.write(small, k, v, near, n, starts)
    assert torch.equal(kv_cache.attend(q, small, near, n), y)


@pytest.mark.parametrize('held', [torch.bfloat16, torch.int8])
def test_steps_captured(gpu, held):
    """A decode step (write, attend) captured once and replayed over other tokens, lengths and pages,
    beside a second graph of the same shapes."""
    lengths = [30, 700, 16]
    table, pages = table_of([n + 8 for n in lengths], 16, torch.Generator().manual_seed(6), 'cuda')
    cache = filled(held, pages, 16, 2, 128, torch.bfloat16)
    mirror = KVCache(*(t.clone() if t is not None else None
                       for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    q = torch.zeros((3, 8, 128), dtype=torch.bfloat16, device='cuda')
    k, v = (torch.zeros((3, 2, 128), dtype=torch.bfloat16, device='cuda') for _ in range(2))
    out, out2 = torch.zeros_like(q), torch.zeros_like(q)

    def step(o):
        kv_cache.write(cache, k, v, table, n)
        kv_cache.attend(q, cache, table, n, out=o)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(out)
        graphs = []
        for o in (out, out2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step(o)
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for t in ('k', 'v', 'k_scale', 'v_scale'):
        if getattr(cache, t) is not None:
            getattr(cache, t).copy_(getattr(mirror, t))
    for i in range(4):
        g = torch.Generator().manual_seed(20 + i)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g).bfloat16())
        n.copy_(torch.tensor([m + i + 1 for m in lengths], dtype=torch.int32))
        kv_cache.write(mirror, k, v, table, n)
        want = kv_cache.attend(q, mirror, table, n)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal((out, out2)[i % 2], want)
        same(cache, mirror)


def test_no_sequences(gpu):
    cache = KVCache.allocate(2, 16, 2, 64)
    table = torch.zeros((0, 1), dtype=torch.int32, device='cuda')
    n = torch.zeros(0, dtype=torch.int32, device='cuda')
    q = torch.zeros((0, 4, 64), dtype=torch.float16, device='cuda')
    assert kv_cache.attend(q, cache, table, n).shape == (0, 4, 64)
    kv_cache.write(cache, q[:, :2], q[:, :2], table, n)
    one = torch.zeros(1, dtype=torch.int32, device='cuda')
    k, v = kv_cache.read(cache, table, one, 5)
    assert k.shape == (5, 2, 64) and not bool(k.any()) and not bool(v.any())
