"""Every way that the host launches the attention over a paged cache, the moves of
its rows and the attention of packed rows, against 64 bits (tolerances: attention_refs).
Which way a call takes is told by the size of its workspace (on 256 CUs)."""
import pytest
import torch

from attention_refs import quantize64, starts_of, table_of
from test_gpu_kv_cache import TYPES, attend_case, check_attend, filled, kv_rows
from test_gpu_packed_attention import run
from w8a8 import _abi, kv_cache
from w8a8.kv_cache import KVCache
from w8a8.packed_attention import packed_attention

pytestmark = pytest.mark.gpu


def route(sequences, heads, kv, dim, keys):
    """None (a workgroup for each pair), or the ranges for each pair that the join's launch goes by."""
    size = _abi.load().w8a8_cache_attend_workspace_size(sequences, heads, kv, dim, keys)
    padded = 64 if dim <= 64 else 128 if dim <= 128 else 256
    pairs = sequences * kv * -(-(heads // kv) // 16)
    return size // (2 * 16 * (padded + 2) * 4 + 16) // pairs if size else None


def lengths_to(most, count, seed):
    g = torch.Generator().manual_seed(seed)
    return [most] + torch.randint(1, most + 1, (count - 1,), generator=g).tolist()


@pytest.mark.parametrize('held,dtype', TYPES)
@pytest.mark.parametrize('dim', [64, 80, 128, 256])
@pytest.mark.parametrize('heads,kv,most,count,each', [
    (4, 2, 700, 6, 6),       # six ranges for each pair: joined range by range
    (28, 28, 1501, 7, 2),    # more pairs than that many ranges fit
    (34, 2, 1000, 3, 8),     # 17 query heads of a key head; joined pair by pair, by four waves
    (8, 1, 9000, 2, 71),     # by eight
    (16, 16, 1100, 40, 0),   # more pairs than workgroups
])
def test_joined_sums(gpu, held, dtype, dim, heads, kv, most, count, each):
    found = route(count, heads, kv, dim, -(-most // 16) * 16)
    assert found == each or (dim == 256 and each == 2 and found == 1)
    attend_case(held, dtype, 16, heads, kv, dim, lengths_to(most, count, dim), seed=dim)


@pytest.mark.parametrize('held,dtype', TYPES)
@pytest.mark.parametrize('dim', [64, 128, 256])
def test_whole_pairs_of_many_blocks(gpu, held, dtype, dim):
    assert route(8, 16, 16, dim, 1024) is None
    attend_case(held, dtype, 64, 16, 16, dim, lengths_to(1024, 8, dim), seed=dim)


@pytest.mark.parametrize('held,dtype', TYPES)
@pytest.mark.parametrize('dim,heads,kv,sequences,width', [
    (64, 16, 8, 3, 3200), (128, 16, 8, 2, 3000), (256, 8, 8, 2, 1500),   # ranges that the lengths leave mostly empty
    (64, 16, 16, 180, 32), (128, 8, 8, 280, 32), (256, 8, 8, 140, 32),   # a workgroup for each pair
])
def test_more_pages_than_the_last_cache_holds(gpu, held, dtype, dim, heads, kv, sequences, width):
    """What the table could name decides how keys are loaded; short contexts in a wide table."""
    page = 32 if width > 32 else 16
    row = dim + 4 if held == torch.int8 else 2 * dim
    scale = 2 if held == torch.int8 else 1
    if width > 32:
        width *= scale
    else:
        sequences *= scale
    assert 2 * row * kv * width * page * sequences > 256 << 20
    assert (route(sequences, heads, kv, dim, width * page) is None) == (width == 32)
    lengths = lengths_to(min(700, width * page), sequences, dim)
    table, pages = table_of(lengths, page, torch.Generator().manual_seed(dim), 'cuda', width=width)
    cache = filled(held, pages, page, kv, dim, dtype, dim)
    q = (torch.randn((sequences, heads, dim), generator=torch.Generator().manual_seed(1)) * 1.5).to(dtype).cuda()
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    y = kv_cache.attend(q, cache, table, n)
    some = slice(0, None, 1 if sequences < 10 else 7)
    check_attend(y[some], q[some], cache, table[some], lengths[some], dim ** -0.5)


@pytest.mark.parametrize('held', [torch.float16, torch.bfloat16, torch.int8])
@pytest.mark.parametrize('dim,heads', [(64, 64), (128, 32), (256, 17)])
def test_moves_of_more_than_the_last_cache_holds(gpu, held, dim, heads):
    dtype = torch.bfloat16 if held == torch.int8 else held
    new, page = [2100, 0, 1, 2099], 64
    assert sum(new) * heads * dim * 4 > 64 << 20
    table, pages = table_of(new, page, torch.Generator().manual_seed(dim), 'cuda')
    cache = KVCache.allocate(pages, page, heads, dim, dtype=held)
    st, starts = starts_of(new, 'cuda')
    k, v = kv_rows(dtype, st[-1] + 3, heads, dim)
    kv_cache.write(cache, k, v, table, torch.tensor(new, dtype=torch.int32, device='cuda'), starts)
    b = torch.repeat_interleave(torch.arange(4), torch.tensor(new))
    key = (torch.arange(st[-1]) - torch.tensor(st)[b]).cuda()
    at = table[b.cuda(), key // page].long()
    back = kv_cache.read(cache, table, starts, st[-1] + 3, dtype=dtype)
    for name, x, y in (('k', k[:-3], back[0]), ('v', v[:-3], back[1])):
        got = getattr(cache, name)[at, :, key % page]
        if held == torch.int8:
            codes, scale = quantize64(x)
            assert torch.equal(got, codes) and torch.equal(getattr(cache, name + '_scale')[at, :, key % page], scale)
            x = (codes.float() * scale[..., None]).to(dtype)
        else:
            assert torch.equal(got, x)
        assert torch.equal(y[:-3], x) and not bool(y[-3:].any())
    used = torch.zeros((pages, page), dtype=torch.bool, device='cuda')
    used[at, key % page] = True
    assert not bool(cache.k.transpose(1, 2)[~used].any()) and not bool(cache.v.transpose(1, 2)[~used].any())


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('dtype,dim', [(torch.float16, 64), (torch.bfloat16, 80), (torch.float16, 96), (torch.bfloat16, 96),
                                       (torch.float16, 128), (torch.float16, 256), (torch.bfloat16, 256)])
@pytest.mark.parametrize('new,keys', [([16], [4000]), ([3, 40], [2500, 2600])])
def test_keys_shared_by_workgroups(gpu, new, keys, dtype, dim, causal):
    assert _abi.load().w8a8_packed_attention_workspace_size(sum(new), sum(keys), len(new), 4, 2, dim) > 0
    run(dtype, 4, 2, dim, new, keys, causal, seed=dim)


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('sequences,rows,keys', [(4, 1500, 1700), (9, 1500, 1700), (4, 40, 6000), (9, 40, 6000)])
def test_packed_starts_out_of_range_stay_in_bounds(gpu, sequences, rows, keys, causal):
    """Whatever starts hold, only the output's rows are written; few sequences, a search, and keys
    that workgroups share. (That the inputs are read within their rows is seen on the CPU: test_packed_tiles.)"""
    heads, dim = 4, 64
    assert (_abi.load().w8a8_packed_attention_workspace_size(rows, keys, sequences, heads, 2, dim) > 0) == (rows == 40)
    big = torch.full((rows + 400, heads, dim), 7.0, dtype=torch.float16, device='cuda')
    q = torch.zeros((rows, heads, dim), dtype=torch.float16, device='cuda')
    k = torch.zeros((keys, 2, dim), dtype=torch.float16, device='cuda')
    low, high = -2 ** 31, 2 ** 31 - 1
    g = torch.Generator().manual_seed(sequences + rows)
    pool = torch.tensor([low, high, -1, 0, 1, rows - 1, rows, rows + 1, keys, keys + 1, 90000, rows // 2])
    for _ in range(8):
        st, ks = (pool[torch.randint(0, len(pool), (sequences + 1,), generator=g)].int().cuda() for _ in range(2))
        for starts, k_starts in ((st, ks), (st.sort().values, ks.sort().values)):
            packed_attention(q, k, k, starts, k_starts, causal=causal, out=big[200:200 + rows])
            packed_attention(q, k, k, starts, k_starts, causal=causal)
    assert bool((big[:200] == 7.0).all()) and bool((big[200 + rows:] == 7.0).all())
