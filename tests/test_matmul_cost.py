"""What the launches of a product are chosen by, compiled for the host: no size that is accepted runs over."""

import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "lplb_b200" / "csrc"
SOURCE = """
#include "matmul_cost.h"
extern "C" long long few(long long tiles, long long fit, int blocks, int cols, int split) { return lplb::ops::few_cycles(tiles, fit, blocks, cols, split); }
extern "C" long long pairs(long long rows, int step, int most, long long tiles_p, long long k_blocks, int n_sm, int* steps) {
  const auto best = lplb::ops::pair_cost(rows, step, most, tiles_p, k_blocks, n_sm);
  *steps = best.steps;
  return best.cycles;
}
"""


@pytest.fixture(scope="module")
def cost(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no compiler")
    at = tmp_path_factory.mktemp("cost")
    (at / "cost.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC), str(at / "cost.cpp"), "-o", str(at / "cost.so")], check=True)
    lib = ctypes.CDLL(str(at / "cost.so"))
    lib.few.restype = lib.pairs.restype = ctypes.c_longlong
    lib.few.argtypes = [ctypes.c_longlong, ctypes.c_longlong, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    lib.pairs.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int, ctypes.c_longlong, ctypes.c_longlong, ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    return lib


def _few(tiles, fit, blocks, cols, split):
    return -(-tiles // fit) * (blocks * (256 + 2 * cols) + 10 * cols + (1500 + 2 * cols if split > 1 else 0))


def test_few_rows_of_the_longest_sum(cost):
    k_blocks = 2**28 // 64
    for m in (1, 112, 113, 128, 256):
        cols = -(-m // 16) * 16
        found = [cost.few(1, 148 // split, -(-k_blocks // split), cols, split) for split in range(1, 9)]
        assert found == [_few(1, 148 // split, -(-k_blocks // split), cols, split) for split in range(1, 9)]
        assert min(found) > 0 and found.index(min(found)) == 7  # dealt out as far as can be


def test_few_rows(cost):
    rng = random.Random(0)
    for _ in range(500):
        args = rng.randint(1, 2**31), rng.randint(1, 148), rng.randint(1, 2**22), 16 * rng.randint(1, 16), rng.randint(1, 8)
        if _few(*args) < 2**63:
            assert cost.few(*args) == _few(*args)


@pytest.mark.parametrize("rows,k_blocks", [(1, 1), (32, 7), (33, 2**22), (1000, 1), (2048, 2**22), (2**31 - 256, 1), (2**31 - 256, 16)])
def test_pairs(cost, rows, k_blocks):
    steps = ctypes.c_int()
    for most in (128, 256):
        cycles = cost.pairs(rows, 32, most, 3, k_blocks, 148, ctypes.byref(steps))
        assert cycles >= k_blocks * 256 and 1 <= steps.value <= most // 32
