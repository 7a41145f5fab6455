"""The tiles of packed sequences, their own header run on the CPU lane by lane, with
nothing readable around the starts: every row is in one tile of its sequence, and
whatever the starts hold, no tile reaches outside of the rows and keys."""
import random
import subprocess
from pathlib import Path

import pytest

import build_lib

TESTS = Path(__file__).resolve().parent
TILE = 128


@pytest.fixture(scope='module')
def find(tmp_path_factory):
    exe = tmp_path_factory.mktemp('tiles') / 'driver'
    subprocess.run(['g++', '-std=c++17', '-O1', '-pthread', f'-I{build_lib.CSRC}', str(TESTS / 'packed_tiles_driver.cpp'),
                    '-o', str(exe)], check=True)

    def run(rows, keys, group, starts, k_starts, side):
        line = ' '.join(map(str, (rows, keys, len(starts) - 1, group, side, *starts, *k_starts)))
        res = subprocess.run([str(exe)], input=line + '\n', text=True, capture_output=True,
                             timeout=60)
        assert res.returncode == 0, f'status {res.returncode}'
        out = res.stdout.splitlines()
        assert int(out[0]) == len(out) - 1
        return [tuple(map(int, x.split())) for x in out[1:]]
    return run


def starts_of(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


@pytest.mark.parametrize('side', [0, 1])
@pytest.mark.parametrize('group', [1, 3, 8])
@pytest.mark.parametrize('sequences', [0, 1, 2, 7, 8, 9, 63, 64, 65, 300])
def test_every_row_is_in_one_tile(find, sequences, group, side):
    rng = random.Random(sequences * 10 + group)
    new = [rng.choice([0, 1, 15, 16, 17, 43, 128, 200]) if sequences < 60 else rng.randrange(6) for _ in range(sequences)]
    starts, k_starts = starts_of(new), starts_of([n + rng.randrange(3) for n in new])
    rows, keys = starts[-1] + 77, k_starts[-1] + 5
    seen = [0] * (rows * group)
    for b, first, n, row0, key0, nk in find(rows, keys, group, starts, k_starts, side):
        if b < 0:
            continue
        assert row0 == starts[b] and first % TILE == 0 and first < n
        assert n == ((rows if b == sequences else starts[b + 1]) - starts[b]) * group
        assert (key0, nk) == ((0, 0) if b == sequences else (k_starts[b], k_starts[b + 1] - k_starts[b])) or nk == 0
        for r in range(row0 * group + first, row0 * group + min(first + TILE, n)):
            seen[r] += 1
    assert set(seen) == {1}


@pytest.mark.parametrize('side', [0, 1])
@pytest.mark.parametrize('sequences', [1, 4, 7, 8, 20, 70])
def test_starts_out_of_range_stay_in_bounds(find, sequences, side):
    rng = random.Random(sequences)
    low, high = -2 ** 31, 2 ** 31 - 1
    for group in (1, 7):
        rows, keys = 150, 260
        for _ in range(6):
            pool = [low, high, -1, 0, 1, 149, 150, 151, 260, 261, 90000, rng.randrange(150), rng.randrange(300)]
            starts, k_starts = ([rng.choice(pool) for _ in range(sequences + 1)] for _ in range(2))
            for b, first, n, row0, key0, nk in find(rows, keys, group, starts, k_starts, side):
                assert -1 <= b <= sequences
                if b >= 0:
                    assert 0 <= row0 and 0 <= first < n and n % group == 0 and row0 + n // group <= rows
                    assert 0 <= key0 and 0 <= nk and key0 + nk <= keys
