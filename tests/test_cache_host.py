"""The paged cache and the attention over packed rows without a GPU: argument
checks of the C entry points (nothing is launched) and of the cache's handle."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from w8a8 import _abi, kv_cache
from w8a8.kv_cache import KVCache
from w8a8.packed_attention import packed_attention


def _status(name, args):
    lib = _abi.load()
    args.struct_size = ctypes.sizeof(args)
    return getattr(lib, name)(ctypes.byref(args)), lib.w8a8_last_error().decode()


def _refused(name, args, fragment):
    rc, message = _status(name, args)
    assert rc == _abi.ERR_INVALID and fragment in message, message


def test_struct_layouts():
    lib = _abi.load()
    assert ctypes.sizeof(_abi.KvCache) == 96
    assert [ctypes.sizeof(s) for s in _abi.CACHE_STRUCTS] == [216, 216, 232, 192]
    for i, st in enumerate(_abi.CACHE_STRUCTS):
        assert lib.w8a8_struct_size(12 + i) == ctypes.sizeof(st)
    for name, st in zip(_abi.CACHE_ENTRY_POINTS, _abi.CACHE_STRUCTS):
        a = st(struct_size=8)
        assert getattr(lib, name)(ctypes.byref(a)) == _abi.ERR_INVALID
        assert 'struct_size' in lib.w8a8_last_error().decode()
        assert getattr(lib, name)(None) == _abi.ERR_INVALID


CACHE = dict(k=1 << 30, v=2 << 30, pages=10, strides=(2 * 16 * 64, 16 * 64, 64), dtype=_abi.F16, page_size=16, heads=2,
             dim=64)
CODES = dict(CACHE, dtype=_abi.I8, k_scale=3 << 30, v_scale=4 << 30, scale_strides=(32, 16))

BAD_CACHES = [
    (dict(dtype=_abi.F32), 'cache dtype'),
    (dict(k=None), 'null'),
    (dict(v=(2 << 30) + 8), 'misaligned'),
    (dict(dim=60), 'dim'), (dict(dim=0), 'dim'), (dict(dim=264), 'dim'),
    (dict(heads=0), 'heads'), (dict(pages=0), 'pages'), (dict(pages=1 << 31), 'pages'),
    (dict(page_size=0), 'page_size'), (dict(page_size=24), 'page_size'), (dict(page_size=4112), 'page_size'),
    (dict(strides=(2048, 1024, 60)), 'strides'), (dict(strides=(2048, 1024, 56)), 'strides'),
    (dict(strides=(-2048, 1024, 64)), 'strides'), (dict(strides=(2048, 1024, 1 << 26)), 'strides'),
]
BAD_CODES = [(dict(k_scale=None), 'scale'), (dict(v_scale=(4 << 30) + 4), 'scale'), (dict(scale_strides=(30, 16)), 'scale'),
             (dict(scale_strides=(32, -16)), 'scale')]

WRITE = dict(dtype=_abi.F16, k=5 << 30, v=6 << 30, k_strides=(128, 64), v_strides=(128, 64), rows=7, sequences=3,
             page_table=7 << 30, ld_table=4, table_width=4, lengths=8 << 30, starts=9 << 30)
READ = {k: v for k, v in WRITE.items() if k != 'lengths'}
ATTEND = dict(dtype=_abi.F16, q=5 << 30, out=6 << 30, q_strides=(512, 64), out_strides=(512, 64), sequences=3, heads=8,
              page_table=7 << 30, ld_table=4, table_width=4, lengths=8 << 30, sm_scale=0.1, workspace=9 << 30,
              workspace_bytes=1 << 30)

LONG = dict(ld_table=1000, table_width=1000)   # keys that several workgroups share


def _args(which, change=None, cache=None, codes=False):
    struct, base = {'write': (_abi.CacheWriteArgs, WRITE), 'read': (_abi.CacheReadArgs, READ),
                    'attend': (_abi.CacheAttendArgs, ATTEND)}[which]
    return struct(cache=_abi.KvCache(**{**(CODES if codes else CACHE), **(cache or {})}), **{**base, **(change or {})})


@pytest.mark.parametrize('which', ['write', 'read', 'attend'])
def test_cache_refusals(which):
    for change, fragment in BAD_CACHES:
        _refused(f'w8a8_cache_{which}', _args(which, cache=change), fragment)
    for change, fragment in BAD_CODES:
        _refused(f'w8a8_cache_{which}', _args(which, cache=change, codes=True), fragment)
    _refused(f'w8a8_cache_{which}', _args(which, dict(dtype=_abi.F32)), 'dtype')
    _refused(f'w8a8_cache_{which}', _args(which, dict(dtype=_abi.BF16)), 'own dtype')
    _refused(f'w8a8_cache_{which}', _args(which, dict(page_table=None)), 'page table')
    _refused(f'w8a8_cache_{which}', _args(which, dict(ld_table=3)), 'page table')
    _refused(f'w8a8_cache_{which}', _args(which, dict(table_width=1 << 23, ld_table=1 << 23)), '2^27')
    _refused(f'w8a8_cache_{which}', _args(which, dict(sequences=-1)), 'sequences')
    _refused(f'w8a8_cache_{which}', _args(which, dict(sequences=1 << 20)), 'sequences')


@pytest.mark.parametrize('change,fragment', [
    (dict(k=None), 'k null'), (dict(v=(6 << 30) + 8), 'v null or misaligned'), (dict(k_strides=(132, 64)), 'k strides'),
    (dict(v_strides=(128, -64)), 'v strides'), (dict(rows=-1), 'rows'), (dict(rows=1 << 31), 'rows'),
])
def test_row_refusals(change, fragment):
    _refused('w8a8_cache_write', _args('write', change), fragment)
    _refused('w8a8_cache_read', _args('read', change), fragment)


def test_write_and_read_refusals():
    _refused('w8a8_cache_write', _args('write', dict(lengths=None)), 'lengths')
    _refused('w8a8_cache_write', _args('write', dict(starts=None)), 'one row')
    _refused('w8a8_cache_write', _args('write', dict(rows=(1 << 31) - 1), dict(heads=65536)), 'too many rows')
    _refused('w8a8_cache_read', _args('read', dict(starts=None)), 'starts')
    for st in ((64, 64), (0, 64), (128, 0), (128, 56)):
        _refused('w8a8_cache_read', _args('read', dict(k_strides=st)), 'overlap')
        _refused('w8a8_cache_read', _args('read', dict(v_strides=st)), 'overlap')
    # rows in the cache's own memory, and outputs in each other's
    for which in ('write', 'read'):
        _refused(f'w8a8_cache_{which}', _args(which, dict(k=(1 << 30) + 2048)), 'overlap the cache')
        _refused(f'w8a8_cache_{which}', _args(which, dict(v=(2 << 30) - 512)), 'overlap the cache')
    _refused('w8a8_cache_read', _args('read', dict(v=(5 << 30) + 64)), 'overlap')
    for which in ('write', 'read'):
        assert _status(f'w8a8_cache_{which}', _args(which, dict(rows=0)))[0] == _abi.OK


@pytest.mark.parametrize('change,codes,ok', [
    ({}, False, True),
    (dict(v=1 << 30), False, False),                                                    # k's own memory
    (dict(v=(1 << 30) + 128, strides=(4096, 2048, 128)), False, True),                  # columns of a token's row
    (dict(v=(1 << 30) + 112, strides=(4096, 2048, 128)), False, False),
    (dict(v=(1 << 30) + 2048, strides=(4096, 2048, 64)), False, True),                  # behind k's tokens of a head
    (dict(v=(1 << 30) + 2032, strides=(4096, 2048, 64)), False, False),
    (dict(v=(1 << 30) + 4096, strides=(4096, 1024, 64)), False, True),                  # behind k's heads of a page
    (dict(v=(1 << 30) + 4096, strides=(2048, 1024, 64)), False, False),
    (dict(v=(1 << 30) + 9 * 4096, strides=(2048, 1024, 64)), False, False),             # k's last page
    (dict(v=(1 << 30) + 10 * 4096, strides=(2048, 1024, 64)), False, True),
    (dict(v=(1 << 30) - 10 * 4096, strides=(2048, 1024, 64)), False, True),
    (dict(v=(1 << 30) - 10 * 4096 + 16, strides=(2048, 1024, 64)), False, False),
    (dict(strides=(2048, 64, 128)), False, True),                                       # tokens before heads
    (dict(strides=(1024, 10240, 64)), False, True),                                     # heads before pages
    (dict(strides=(0, 1024, 64)), False, False),                                        # one page, many times
    (dict(strides=(2048, 0, 64)), False, False),
    (dict(strides=(1024, 1024, 64)), False, False),
    (dict(strides=(2048, 1016, 64)), False, False),
    (dict(strides=(0, 1024, 64), pages=1), False, True),                                # (steps that are not taken)
    (dict(strides=(1024, 0, 64), heads=1, dim=64), False, True),
    ({}, True, True),
    (dict(v_scale=3 << 30), True, False),
    (dict(v_scale=(3 << 30) + 64, scale_strides=(64, 32)), True, True),
    (dict(v_scale=(3 << 30) + 48, scale_strides=(64, 32)), True, False),
    (dict(scale_strides=(16, 16)), True, False),
])
def test_places_that_share_memory_are_not_written(change, codes, ok):
    """(Of no sequences, so that what is not refused launches nothing.)"""
    args = _args('write', dict(sequences=0), change, codes)
    if 'heads' in change:
        args.k_strides = args.v_strides = (64, 64)
    rc, message = _status('w8a8_cache_write', args)
    assert rc == (_abi.OK if ok else _abi.ERR_INVALID) and (ok or 'share memory' in message), message


@pytest.mark.parametrize('change,ok', [
    # codes of 2 heads, 16 tokens of 64 (2048 bytes a page), scales of 64 bytes a head
    (dict(k_scale=1 << 30), False),                                                     # in k's own pages
    (dict(v_scale=(1 << 30) + 1024), False),
    (dict(k_scale=(2 << 30) + 9 * 2048 + 2032), False),                                 # v's last codes
    (dict(k_scale=(2 << 30) + 10 * 2048), True),                                        # behind them
    (dict(k_scale=(2 << 30) - (9 * 128 + 128)), True),                                  # before the first
    (dict(k_scale=(2 << 30) - (9 * 128 + 112)), False),
    # a page's codes, then its scales
    (dict(strides=(2048 + 128, 1024, 64), k_scale=(1 << 30) + 2048, scale_strides=(544, 16),
          v_scale=(2 << 30) + 2048), True),
    (dict(strides=(2048 + 128, 1024, 64), k_scale=(1 << 30) + 2032, scale_strides=(544, 16),
          v_scale=(2 << 30) + 2048), False),
    (dict(strides=(2048 + 128, 1024, 64), k_scale=(1 << 30) + 2048, scale_strides=(544, 16),
          v_scale=(2 << 30) + 2064), False),                                            # the next page's codes
    (dict(strides=(2048 + 128, 1024, 64), k_scale=(1 << 30) + 2048, scale_strides=(548, 16),
          v_scale=(2 << 30) + 2048), False),                                            # steps of another length
    # a head's codes, then its scales
    (dict(strides=(2 * 1088, 1088, 64), k_scale=(1 << 30) + 1024, scale_strides=(544, 272),
          v_scale=(2 << 30) + 1024), True),
    (dict(strides=(2 * 1088, 1088, 64), k_scale=(1 << 30) + 1008, scale_strides=(544, 272),
          v_scale=(2 << 30) + 1024), False),
    (dict(strides=(2 * 1088, 1088, 64), k_scale=(1 << 30) + 1024, scale_strides=(544, 272),
          v_scale=(2 << 30) + 1040), False),
    # heads before pages
    (dict(strides=(1088, 10 * 1088, 64), k_scale=(1 << 30) + 1024, scale_strides=(272, 2720),
          v_scale=(2 << 30) + 1024), True),
    (dict(strides=(1088, 10 * 1088, 64), k_scale=(1 << 30) + 1024, scale_strides=(272, 2720),
          v_scale=(2 << 30) + 1040), False),
    # tokens before heads, a page's scales behind its codes
    (dict(strides=(2176, 64, 128), k_scale=(1 << 30) + 2048, scale_strides=(544, 16), v_scale=(2 << 30) + 2048), True),
    (dict(strides=(2176, 64, 128), k_scale=(1 << 30) + 2016, scale_strides=(544, 16), v_scale=(2 << 30) + 2048), False),
    # one page, whose step is not taken
    (dict(pages=1, strides=(0, 1088, 64), k_scale=(1 << 30) + 1024, scale_strides=(4, 272), v_scale=(2 << 30) + 1024), True),
    # k, v and both scales in one page
    (dict(v=(1 << 30) + 2048, strides=(4352, 1024, 64), k_scale=(1 << 30) + 4096, scale_strides=(1088, 16),
          v_scale=(1 << 30) + 4224), True),
    (dict(v=(1 << 30) + 2048, strides=(4352, 1024, 64), k_scale=(1 << 30) + 4096, scale_strides=(1088, 16),
          v_scale=(1 << 30) + 4352), False),
])
def test_codes_and_scales_that_share_memory_are_not_written(change, ok):
    rc, message = _status('w8a8_cache_write', _args('write', dict(sequences=0), change, True))
    assert rc == (_abi.OK if ok else _abi.ERR_INVALID) and (ok or 'share memory' in message), message


@pytest.mark.parametrize('scale', [3 << 30, 4 << 30])
def test_rows_over_scales_are_refused(scale):
    """10 pages of 2 heads of 16 scales: 1280 bytes."""
    for at in (scale, scale + 1264, scale - 512):
        for which in ('write', 'read'):
            for name in ('k', 'v'):
                _refused(f'w8a8_cache_{which}', _args(which, {name: at}, codes=True), 'overlap the cache')
        _refused('w8a8_cache_attend', _args('attend', dict(out=at), codes=True), 'out overlaps the cache')
    for which in ('write', 'read'):   # behind them (the next refusal is another)
        missing, fragment = (dict(lengths=None), 'lengths') if which == 'write' else (dict(starts=None), 'starts')
        _refused(f'w8a8_cache_{which}', _args(which, {'k': scale + 1280, **missing}, codes=True), fragment)
    _refused('w8a8_cache_attend', _args('attend', dict(out=scale + 1280, lengths=None), codes=True), 'lengths')


def test_integers_in_what_is_written_are_refused():
    """Tables, lengths and starts that a kernel would write over while it reads them, and workspaces."""
    none = dict(sequences=0)   # (launches nothing where it is not refused)
    for codes, at in ((False, 1 << 30), (False, (2 << 30) + 40000), (True, (1 << 30) + 640), (True, 3 << 30), (True, (4 << 30) + 1276)):
        for name in ('page_table', 'lengths', 'starts'):
            _refused('w8a8_cache_write', _args('write', {name: at}, codes=codes), 'lie in the cache')
    assert _status('w8a8_cache_write', _args('write', dict(none, starts=(2 << 30) + 40960)))[0] == _abi.OK
    assert _status('w8a8_cache_write', _args('write', dict(none, starts=(1 << 30) - 4)))[0] == _abi.OK
    # in the gaps between the pages' rows, and across them
    gaps = dict(strides=(4096, 1024, 64))
    assert _status('w8a8_cache_write', _args('write', dict(none, starts=(1 << 30) + 4096), gaps))[0] == _abi.OK
    _refused('w8a8_cache_write', _args('write', dict(none, starts=(1 << 30) + 4092), gaps), 'lie in the cache')
    for at in (5 << 30, (6 << 30) + 7 * 256 - 4):
        for name in ('page_table', 'starts'):
            _refused('w8a8_cache_read', _args('read', {name: at}), 'lie in an output')
    for name in ('page_table', 'lengths'):
        for at in (6 << 30, (6 << 30) + 3 * 1024 - 4, (6 << 30) - 8):
            _refused('w8a8_cache_attend', _args('attend', {name: at}), 'lie in the output')
    _refused('w8a8_cache_attend', _args('attend', dict(workspace=(6 << 30) - 16, **LONG)), 'lie in the output')
    for change in (dict(starts=4 << 30), dict(k_starts=(4 << 30) - 8), dict(starts=(4 << 30) + 100 * 512 - 4)):
        _refused('w8a8_packed_attention', _abi.PackedAttentionArgs(**{**PACKED, **change}), 'lie in the output')
    few = dict(rows=16, keys=4000, sequences=1, workspace_bytes=1 << 30)
    assert _abi.load().w8a8_packed_attention_workspace_size(16, 4000, 1, 4, 2, 64) > 0
    _refused('w8a8_packed_attention', _abi.PackedAttentionArgs(**{**PACKED, **few, 'workspace': (4 << 30) - 16}), 'lie in the output')


@pytest.mark.parametrize('change,fragment', [
    (dict(q=None), 'q null'), (dict(out=(6 << 30) + 8), 'out null or misaligned'), (dict(q_strides=(516, 64)), 'q strides'),
    (dict(out_strides=(512, 0)), 'overlap'), (dict(out_strides=(448, 64)), 'overlap'), (dict(out=5 << 30), 'overlaps q'),
    (dict(out=(2 << 30) + 64), 'overlaps the cache'),
    (dict(heads=0), 'heads'), (dict(heads=7), 'heads'), (dict(heads=65538), 'heads'), (dict(lengths=None), 'lengths'),
    (dict(sm_scale=0.0), 'sm_scale'), (dict(sm_scale=-1.0), 'sm_scale'), (dict(sm_scale=float('inf')), 'sm_scale'),
    (dict(sm_scale=float('nan')), 'sm_scale'), (dict(workspace=None, **LONG), 'workspace'), (dict(workspace_bytes=64, **LONG), 'workspace'),
    (dict(workspace=(9 << 30) + 4, **LONG), 'workspace'),
])
def test_attend_refusals(change, fragment):
    _refused('w8a8_cache_attend', _args('attend', change), fragment)


def test_attend_workspace():
    lib = _abi.load()
    assert lib.w8a8_cache_attend_workspace_size(0, 8, 2, 64, 100) == 0
    assert lib.w8a8_cache_attend_workspace_size(3, 8, 3, 64, 100) == 0
    small, large = (lib.w8a8_cache_attend_workspace_size(1, 8, 2, 128, n) for n in (100, 1 << 20))
    assert 0 <= small <= large < 1 << 26
    assert lib.w8a8_cache_attend_workspace_size(100000, 64, 8, 128, 1 << 26) == large
    assert _status('w8a8_cache_attend', _args('attend', dict(sequences=0)))[0] == _abi.OK


PACKED = dict(dtype=_abi.F16, q=1 << 30, k=2 << 30, v=3 << 30, out=4 << 30, q_strides=(256, 64), k_strides=(128, 64),
              v_strides=(128, 64), out_strides=(256, 64), rows=100, keys=120, sequences=2, heads=4, kv_heads=2, dim=64,
              causal=1, starts=5 << 30, k_starts=6 << 30, sm_scale=0.1)


@pytest.mark.parametrize('change,fragment', [
    (dict(dtype=_abi.F32), 'dtype'), (dict(dim=60), 'dim'), (dict(dim=264), 'dim'), (dict(dim=0), 'dim'),
    (dict(heads=0), 'heads'), (dict(heads=5), 'heads'), (dict(kv_heads=0), 'heads'), (dict(heads=65538), 'heads'),
    (dict(rows=-1), 'rows'), (dict(rows=1 << 27), 'rows'), (dict(keys=1 << 27), 'keys'), (dict(keys=-1), 'keys'),
    (dict(sequences=1 << 20), 'sequences'), (dict(sequences=-1), 'sequences'), (dict(sm_scale=0.0), 'sm_scale'),
    (dict(sm_scale=float('inf')), 'sm_scale'), (dict(causal=2), 'causal'), (dict(q=None), 'q null'),
    (dict(k=(2 << 30) + 8), 'k null or misaligned'), (dict(v=None), 'v null'), (dict(out=None), 'out null'),
    (dict(q_strides=(260, 64)), 'q strides'), (dict(k_strides=(128, -8)), 'k strides'), (dict(k_strides=(56, 64)), 'row strides'),
    (dict(v_strides=(1 << 23, 64)), 'row strides'), (dict(starts=None), 'starts'), (dict(k_starts=None), 'starts'),
    (dict(out_strides=(192, 64)), 'output rows overlap'), (dict(out_strides=(256, 0)), 'output rows overlap'),
    (dict(out=1 << 30), 'overlaps an input'), (dict(out=(2 << 30) - 64), 'overlaps an input'),
    (dict(out=(3 << 30) + 16), 'overlaps an input'), (dict(rows=(1 << 27) - 1, heads=64, kv_heads=64, q_strides=(4096, 64),
                                                           out_strides=(4096, 64), out=1 << 44), 'too many'),
])
def test_packed_attention_refusals(change, fragment):
    _refused('w8a8_packed_attention', _abi.PackedAttentionArgs(**{**PACKED, **change}), fragment)


def test_workspaces_of_sizes_that_are_refused():
    lib = _abi.load()
    good = (1, 4000, 1, 4, 2, 64)
    assert lib.w8a8_packed_attention_workspace_size(*good) > 0
    for i, values in enumerate([(0, -1, 1 << 27, (1 << 63) - 1), (0, -1, 1 << 27, (1 << 63) - 1), (0, -1, 1 << 20, (1 << 63) - 1),
                                (0, -4, 1, 3, 65538, 1 << 62), (0, -2, 3, 8, 1 << 62), (0, -8, 4, 60, 264, (1 << 31) - 1)]):
        for value in values:
            assert lib.w8a8_packed_attention_workspace_size(*good[:i], value, *good[i + 1:]) == 0, (i, value)
    good = (1, 8, 2, 128, 100000)
    assert lib.w8a8_cache_attend_workspace_size(*good) > 0
    for i, values in enumerate([(0, -1, 1 << 20, (1 << 63) - 1), (0, -2, 7, 65538, 1 << 62), (0, -2, 3, 16, 1 << 62),
                                (0, -8, 264, (1 << 31) - 1), (-1, 1 << 27, (1 << 63) - 1)]):
        for value in values:
            assert lib.w8a8_cache_attend_workspace_size(*good[:i], value, *good[i + 1:]) == 0, (i, value)


def test_packed_attention_of_nothing():
    assert _status('w8a8_packed_attention', _abi.PackedAttentionArgs(**{**PACKED, 'rows': 0}))[0] == _abi.OK


# ------------------------------------------------------------- the handle
def _buffers(shape=(3, 2, 16, 64), dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype), torch.zeros(shape, dtype=dtype)


def test_handle():
    k, v = _buffers()
    c = KVCache(k, v)
    assert (c.heads, c.page_size, c.dim, c.codes) == (2, 16, 64, False)
    c = KVCache.allocate(3, 48, 2, 72, dtype=torch.int8, device='cpu')
    assert c.codes and c.k_scale.shape == (3, 2, 48) and c.k.shape == (3, 2, 48, 72)


@pytest.mark.parametrize('shape', [(3, 2, 16), (0, 2, 16, 64), (3, 0, 16, 64), (3, 2, 24, 64), (3, 2, 4112, 64), (3, 2, 16, 60),
                                   (3, 2, 16, 264), (3, 2, 0, 64)])
def test_handles_are_refused(shape):
    with pytest.raises(ValueError):
        KVCache(*_buffers(shape))


def test_handles_of_other_tensors_are_refused():
    k, v = _buffers()
    for a, b in ((k, v.bfloat16()), (k, v[:2]), (k.float(), v.float()), (k, torch.zeros((3, 16, 2, 64)).half().transpose(1, 2)),
                 (k.transpose(2, 3).contiguous().transpose(2, 3),) * 2, (torch.zeros((3, 2, 16, 68)).half()[..., :64],) * 2,
                 (torch.zeros(3 * 2 * 16 * 64 + 4).half()[4:].view(3, 2, 16, 64),) * 2):
        with pytest.raises(ValueError):
            KVCache(a, b)
    s = torch.zeros((3, 2, 16))
    k8, v8 = _buffers(dtype=torch.int8)
    for args in ((k, v, s, s), (k8, v8), (k8, v8, s), (k8, v8, s, s.half()), (k8, v8, s, s[:2]),
                 (k8, v8, s, torch.zeros((3, 16, 2)).transpose(1, 2)), (k8, v8, *(torch.zeros((3, 2, 18))[..., :16],) * 2)):
        with pytest.raises(ValueError):
            KVCache(*args)


def _calls(grad=None, wrap=lambda t: t):
    cache = KVCache(*_buffers())
    table = torch.zeros((1, 1), dtype=torch.int32)
    n, starts = torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    x, q = torch.zeros((1, 2, 64)).half(), torch.zeros((1, 4, 64)).half()
    return {
        'write': lambda: kv_cache.write(cache, wrap(x), x, table, n),
        'write v': lambda: kv_cache.write(cache, x, wrap(x), table, n),
        'read out': lambda: kv_cache.read(cache, table, starts, 1, out=(wrap(x), x)),
        'attend': lambda: kv_cache.attend(wrap(q), cache, table, n),
        'attend out': lambda: kv_cache.attend(q, cache, table, n, out=wrap(q.clone())),
        'packed': lambda: packed_attention(wrap(q), x, x, starts),
        'packed k': lambda: packed_attention(q, wrap(x), x, starts),
        'packed v': lambda: packed_attention(q, x, wrap(x), starts),
        'packed out': lambda: packed_attention(q, x, x, starts, out=wrap(q.clone())),
        'a cache': lambda: kv_cache.attend(q, KVCache(wrap(cache.k), cache.v), table, n),
    }


def test_gradients_are_refused_not_lost():
    for name, call in _calls(wrap=lambda t: t.clone().requires_grad_()).items():
        with pytest.raises(ValueError, match='no gradient'):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match='HIP device'):
            call()


def test_forward_mode_tangents_are_refused():
    with forward_ad.dual_level():
        for name, call in _calls(wrap=lambda t: forward_ad.make_dual(t, torch.ones_like(t))).items():
            with torch.no_grad(), pytest.raises(ValueError, match='no gradient'):
                call()


def test_cpu_tensors_are_refused():
    for name, call in _calls().items():
        with pytest.raises(ValueError, match='HIP device'):
            call()
