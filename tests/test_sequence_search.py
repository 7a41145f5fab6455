"""The search for a packed row's sequence, its own header run on the CPU lane by
lane, with nothing readable around the starts and lengths."""
import subprocess
from pathlib import Path

import pytest

import build_lib

TESTS = Path(__file__).resolve().parent


@pytest.fixture(scope='module')
def search(tmp_path_factory):
    exe = tmp_path_factory.mktemp('sequences') / 'driver'
    subprocess.run(['g++', '-std=c++17', '-O1', '-pthread', f'-I{build_lib.CSRC}', str(TESTS / 'sequence_driver.cpp'),
                    '-o', str(exe)], check=True)

    def run(cases):
        res = subprocess.run([str(exe)], input=''.join('%d %d %d %d\n' % c for c in cases), text=True, capture_output=True,
                             timeout=60)
        assert res.returncode == 0, f'status {res.returncode} after {len(res.stdout.splitlines())} of {len(cases)} cases'
        return [tuple(map(int, line.split())) for line in res.stdout.splitlines()]
    return run


def _want(n, row, lengths):
    at = [(b + 1) // 2 * 3 for b in range(n + 1)]
    for b in range(n):
        if at[b] <= row < at[b + 1]:
            return b, at[b], at[b + 1], 100 + b if lengths else 0
    return n, 0, 0, 0


@pytest.mark.parametrize('n', [0, 1, 2, 63, 64, 65, 127, 128, 129, 1000, 4097])
def test_search_stays_within_the_starts(search, n):
    end = (n + 1) // 2 * 3
    rows = sorted({0, 1, 2, 3, 95, 96, end // 2, max(end - 1, 0), end, end + 1, end + 5000})
    cases = [(n, row, lengths, side) for row in rows for lengths in (0, 1) for side in (0, 1)]
    assert search(cases) == [_want(n, row, lengths) for n, row, lengths, _ in cases]
