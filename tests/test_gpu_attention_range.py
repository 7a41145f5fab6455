"""Attention where weights, values and scores lie far apart, against 64 bits
(tolerances: attention_refs, but for what is said here)."""
import math

import pytest
import torch

from attention_refs import attention64, bound, check, quantize64
from w8a8 import kv_cache
from w8a8.kv_cache import KVCache
from w8a8.packed_attention import packed_attention

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
TABLE_PAGE = 64


def paged(k, v, held):
    """A cache of one sequence's keys and values [keys, heads, dim], and its table and length."""
    n, heads, dim = k.shape
    pages = -(-n // TABLE_PAGE)
    cache = KVCache.allocate(pages, TABLE_PAGE, heads, dim, dtype=held)
    for name, x in (('k', k), ('v', v)):
        full = torch.zeros((pages * TABLE_PAGE, heads, dim), dtype=x.dtype, device='cuda')
        full[:n] = x
        full = full.view(pages, TABLE_PAGE, heads, dim).transpose(1, 2)
        if held == torch.int8:
            c, s = quantize64(full)
            getattr(cache, name).copy_(c)
            getattr(cache, name + '_scale').copy_(s)
        else:
            getattr(cache, name).copy_(full)
    table = torch.arange(pages, dtype=torch.int32, device='cuda')[None]
    return cache, table, torch.tensor([n], dtype=torch.int32, device='cuda')


def rows_of(x, n):
    """A cache's [pages, heads, page, ...] as [keys, heads, ...]."""
    return x.transpose(1, 2).flatten(0, 1)[:n]


def keys_with_scores(q0, t, dim, dtype):
    """Keys [keys, 1, dim] whose scores with q0 (one value in every channel), times
    1 / sqrt(dim), are about t (in powers of 2)."""
    return (t[:, None, None] * math.log(2.0) / (q0 * math.sqrt(dim))).expand(-1, 1, dim).contiguous().to(dtype)


def attend_codes(k, v, v_times, dtype, q):
    """Codes whose scales of v are taken times v_times [keys]; o against 64 bits. What
    the kernel loses of P lies below 2^-32 of the largest product of a weight and a
    value's scale, whatever the scales of keys without weight."""
    n, dim = k.shape[0], k.shape[2]
    cache, table, length = paged(k, v, torch.int8)
    flat = torch.ones(table.shape[1] * TABLE_PAGE, device='cuda')
    flat[:n] = v_times
    cache.v_scale.mul_(flat.view(-1, 1, TABLE_PAGE))
    y = kv_cache.attend(q, cache, table, length)
    ks, vs = rows_of(cache.k_scale, n).double(), rows_of(cache.v_scale, n).double()
    k64, codes = rows_of(cache.k, n)[:, 0].double() * ks, rows_of(cache.v, n)[:, 0].double()
    for h in range(q.shape[1]):
        t = (k64 @ q[0, h].double()) * dim ** -0.5
        most = (torch.exp(t - t.max()) * vs[:, 0]).max()
        lost = codes.abs() * most * 2.0 ** -7   # (the bound takes 2^-25 of it)
        o, parts = attention64(q[0, h][None].double(), k64, codes * vs, dim ** -0.5, codes_scale=lost)
        check(y[0, h][None], o, bound(o, parts, dtype), f'head {h}')


@pytest.mark.parametrize('n', [200, 3000])
@pytest.mark.parametrize('dim', [64, 80, 128, 256])
@pytest.mark.parametrize('dtype', DTYPES)
def test_codes_beside_a_row_of_large_values(gpu, dtype, dim, n):
    """A value row far larger than the others, of a key of little weight."""
    g = torch.Generator().manual_seed(dim)
    q = (1.0 + 0.01 * torch.randn((1, 3, dim), generator=g)).to(dtype).cuda()
    for at in (0, 37, n - 1):
        for size in (0, 10, 18, 26, 40, 46) if dtype == torch.float16 else (0, 18, 26, 46, 60, 90):
            t = torch.randn(n, generator=g)
            t[at] = -46.0
            k = keys_with_scores(1.0, t.cuda(), dim, dtype)
            v = (torch.randn((n, 1, dim), generator=g) * 2.0 ** -10).to(dtype).cuda()
            times = torch.ones(n, device='cuda')
            times[at] = 2.0 ** size
            attend_codes(k, v, times, dtype, q)


@pytest.mark.parametrize('n', [200, 3000])
@pytest.mark.parametrize('order', ['up', 'down', 'any'])
@pytest.mark.parametrize('dim', [64, 128, 256])
def test_codes_whose_scales_undo_their_weights(gpu, dim, order, n):
    """Weights over a range of 2^80, the scales of values over its inverse: all keys contribute alike."""
    g = torch.Generator().manual_seed(dim)
    q = (1.0 + 0.01 * torch.randn((1, 2, dim), generator=g)).bfloat16().cuda()
    t = torch.linspace(-40.0, 40.0, n)
    t = t.flip(0) if order == 'down' else t[torch.randperm(n, generator=g)] if order == 'any' else t
    k = keys_with_scores(1.0, t.cuda(), dim, torch.bfloat16)
    v = torch.randn((n, 1, dim), generator=g).bfloat16().cuda()
    attend_codes(k, v, torch.exp2(-t).cuda(), torch.bfloat16, q)


def test_codes_of_the_largest_values(gpu):
    """The largest finite rows beside rows of zeros and of the smallest scale."""
    g = torch.Generator().manual_seed(5)
    k = torch.randn((150, 1, 64), generator=g).bfloat16().cuda()
    v = torch.randn((150, 1, 64), generator=g).bfloat16().cuda()
    v[::3], v[1::3] = 0.0, torch.finfo(torch.bfloat16).max / 4
    q = torch.randn((1, 4, 64), generator=g).bfloat16().cuda()
    attend_codes(k, v, torch.ones(150, device='cuda'), torch.bfloat16, q)


def held_of(dtype, n, dim, t, v):
    """(q, k, v) of one head: scores of about t (powers of 2) with every query."""
    return keys_with_scores(1.0, t.cuda(), dim, dtype), v.to(dtype).cuda()


def check_tail(y, q, k, v, nq_first, what):
    """y [nq, heads, dim]; query i sees the keys before nq_first[i]. What fp16 loses of P
    lies below 2^-32 of the largest."""
    dim = q.shape[2]
    for h in range(q.shape[1]):
        o, parts = attention64(q[:, h].double(), k[:, 0].double(), v[:, 0].double(), dim ** -0.5, nq_first)
        a, lost, d, nk, codes = parts
        check(y[:, h], o, bound(o, (a, lost * 2.0 ** -7, d, nk, codes), q.dtype), f'{what} head {h}')


@pytest.mark.parametrize('dim', [64, 80, 128, 256])
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('n', [500, 5000])
def test_many_keys_of_little_weight(gpu, dtype, dim, n):
    """One key of nearly all the weight whose value is 0: the others, of weights from
    2^-24 to 2^-30, are what is left."""
    g = torch.Generator().manual_seed(dim)
    q = (1.0 + 0.01 * torch.randn((40, 2, dim), generator=g)).to(dtype).cuda()
    for at in (0, 70, n - 41):
        t = -24.0 - 6.0 * torch.rand(n, generator=g)
        t[at] = 0.0
        v = 100.0 + torch.randn((n, 1, dim), generator=g)
        v[at] = 0.0
        k, v = held_of(dtype, n, dim, t, v)
        cache, table, length = paged(k, v, dtype)
        check_tail(kv_cache.attend(q[:1], cache, table, length), q[:1], k, v, None, 'one token')
        for nq in (1, 40):
            starts, k_starts = (torch.tensor([0, m], dtype=torch.int32, device='cuda') for m in (nq, n))
            for causal in (False, True):
                first = torch.arange(nq, device='cuda') + n - nq + 1 if causal else None
                y = packed_attention(q[:nq], k, v, starts, k_starts, causal=causal)
                check_tail(y, q[:nq], k, v, first, f'{nq} rows, causal {causal}')


@pytest.mark.parametrize('dim', [64, 80, 128, 256])
@pytest.mark.parametrize('n', [300, 5000])
def test_values_near_the_largest(gpu, dim, n):
    """Finite bf16 values whose weighted sum is finite, behind keys of less weight."""
    g = torch.Generator().manual_seed(dim)
    q = (1.0 + 0.01 * torch.randn((40, 2, dim), generator=g)).bfloat16().cuda()
    t = torch.full((n,), -7.5)
    t[n - 45] = 0.0
    v = torch.randn((n, 1, dim), generator=g)
    v[n - 45] = 3e38
    k, v = held_of(torch.bfloat16, n, dim, t, v)
    cache, table, length = paged(k, v, torch.bfloat16)
    check_tail(kv_cache.attend(q[:1], cache, table, length), q[:1], k, v, None, 'one token')
    for nq in (1, 40):
        starts, k_starts = (torch.tensor([0, m], dtype=torch.int32, device='cuda') for m in (nq, n))
        for causal in (False, True):
            first = torch.arange(nq, device='cuda') + n - nq + 1 if causal else None
            y = packed_attention(q[:nq], k, v, starts, k_starts, causal=causal)
            check_tail(y, q[:nq], k, v, first, f'{nq} rows, causal {causal}')


@pytest.mark.parametrize('dim', [64, 80, 128, 256])
@pytest.mark.parametrize('n', [300, 5000])
@pytest.mark.parametrize('dtype', DTYPES)
def test_scores_of_minus_infinity(gpu, dtype, dim, n):
    """Keys with the score -inf have no weight; if a query sees no others it is 0 / 0, and if it sees no key 0."""
    g = torch.Generator().manual_seed(dim)
    q = (1.0 + 0.01 * torch.randn((40, 2, dim), generator=g)).to(dtype).cuda()
    k, v = (torch.randn((n, 1, dim), generator=g).to(dtype).cuda() for _ in range(2))
    k[:, :, 3] = -math.inf
    nq = 40
    starts = torch.tensor([0, nq], dtype=torch.int32, device='cuda')
    k_starts = torch.tensor([0, n], dtype=torch.int32, device='cuda')
    cache, table, length = paged(k, v, dtype)
    assert bool(torch.isnan(kv_cache.attend(q[:1], cache, table, length)).all())
    assert not bool(kv_cache.attend(q[:1], cache, table, length * 0).any())
    assert not bool(kv_cache.attend(q[:1], cache, table * 0 - 1, length).any())
    for causal in (False, True):
        assert bool(torch.isnan(packed_attention(q, k, v, starts, k_starts, causal=causal)).all())
    few = 30   # of 40 queries the first 10 see no key
    y = packed_attention(q, k[:few], v[:few], starts, torch.tensor([0, few], dtype=torch.int32, device='cuda'))
    assert not bool(y[:10].any()) and bool(torch.isnan(y[10:]).all())
    # some keys with a score: those alone count
    seen = torch.zeros(n, dtype=torch.bool)
    seen[torch.tensor([60, n // 2, n - 60])] = True
    k[seen] = torch.randn((3, 1, dim), generator=g).to(dtype).cuda()
    cache, table, length = paged(k, v, dtype)
    o, parts = zip(*(attention64(q[:, h].double(), k[seen][:, 0].double(), v[seen][:, 0].double(), dim ** -0.5) for h in range(2)))
    for h in range(2):
        check(kv_cache.attend(q[:1], cache, table, length)[:, h], o[h][:1],
              bound(o[h], parts[h], dtype)[:1], 'one token')
        for causal in (False, True):
            y = packed_attention(q, k, v, starts, k_starts, causal=causal)
            check(y[:, h], o[h], bound(o[h], parts[h], dtype), f'causal {causal}')


def test_codes_with_scores_of_minus_infinity(gpu):
    """The same of codes, by scales of k that are infinite."""
    q = torch.ones((1, 2, 64), dtype=torch.float16, device='cuda')
    k, v = -torch.ones((300, 1, 64), dtype=torch.float16, device='cuda'), torch.ones((300, 1, 64), dtype=torch.float16, device='cuda')
    for n in (300, 5000):
        cache, table, length = paged(k.repeat(17, 1, 1)[:n], v.repeat(17, 1, 1)[:n], torch.int8)
        cache.k_scale.fill_(math.inf)
        assert bool(torch.isnan(kv_cache.attend(q, cache, table, length)).all())
        assert not bool(kv_cache.attend(q, cache, table, length * 0).any())
        cache.k_scale[0, 0, 7] = 1.0
        check(kv_cache.attend(q, cache, table, length)[0], torch.ones((2, 64), dtype=torch.float64, device='cuda'),
              torch.full((2, 64), 2.0 ** -10, dtype=torch.float64, device='cuda'))
