"""The forms the host picks for products of block-scaled operands (CPU: the header is compiled for the host and called)."""

import ctypes as C
import heapq
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "pypto_amd" / "csrc"

_SOURCE = """
#include "launch_choice.h"
extern "C" void tile(int64_t m, int64_t n, int64_t kb, int exact, int rows, int cols, int splits, int* out) {
  const pto_hip::BlockTile t = pto_hip::choose_block_tile(m, n, kb, exact != 0, 256, rows, cols, splits);
  out[0] = t.rows, out[1] = t.cols, out[2] = t.per_split;
  for (int i = 0; i < 3; ++i) out[3 + i] = t.tiles[i];
}
extern "C" double span(int64_t a, int64_t b, int64_t c, double x, double y, double z, int64_t cus) { return pto_hip::makespan({a, b, c}, {x, y, z}, cus); }
extern "C" int direct(int64_t slots, int64_t experts, int64_t hidden, int64_t inter) { return pto_hip::experts_direct(slots, experts, hidden, inter, false); }
extern "C" int rows(int64_t slots, int64_t experts, int64_t hidden, int64_t inter, int up, int down) {
  return pto_hip::choose_expert_rows(slots, experts, hidden, inter, up != 0, down != 0, 256);
}
"""


@pytest.fixture(scope="module")
def choice(tmp_path_factory):
    d = tmp_path_factory.mktemp("choice")
    (d / "choice.cpp").write_text(_SOURCE)
    so = d / "choice.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(d / "choice.cpp"), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.tile.argtypes = [C.c_int64] * 3 + [C.c_int] * 4 + [C.POINTER(C.c_int)]
    lib.span.argtypes, lib.span.restype = [C.c_int64] * 3 + [C.c_double] * 3 + [C.c_int64], C.c_double
    lib.direct.argtypes = [C.c_int64] * 4
    lib.rows.argtypes = [C.c_int64] * 4 + [C.c_int] * 2
    return lib


def _tile(lib, m, n, kb, exact=False, rows=0, cols=0, splits=0):
    out = (C.c_int * 6)()
    lib.tile(m, n, kb, exact, rows, cols, splits, out)
    if out[1] == 256:  # every tile starts inside the rows, and they hold all of them
        heights = [out[0], out[0] // 2, out[0] // 4]
        last, first = 0, 0
        for tiles, height in zip(out[3:], heights):
            assert tiles >= 0 and (tiles == 0 or height >= 64)
            if tiles:
                last = first + (tiles - 1) * height
                first += tiles * height
        assert last < m <= first
    return tuple(out[:3])


FORMS = {(16, 16), (16, 32), (64, 64), (64, 128), (64, 256), (128, 256), (256, 256)}


def test_every_size_gets_a_form_that_there_is(choice):
    for m in (1, 2, 15, 16, 17, 33, 64, 65, 200, 333, 1000, 4096, 1 << 20, (1 << 24) - 1):
        for n in (1, 16, 100, 4096, 5003, 20000, 1 << 20):
            for kb in (1, 2, 7, 32, 86, 512):
                for exact in (False, True):
                    rows, cols, per = _tile(choice, m, n, kb, exact)
                    assert (rows, cols) in FORMS and (rows > 16 or m <= 16) and not (exact and rows == 256)
                    assert per == 0 or (8 <= per < kb and (kb + per - 1) // per <= 16)
                    # a launch's work items stay below 2^32
                    wgs = -(-m // rows) * -(-n // cols) * (-(-kb // per) if per else 1)
                    assert wgs * 512 < 1 << 32 or m * n > 1 << 34


def test_tiles_of_several_heights_hold_all_rows(choice):
    for m in [*range(1, 1100), 2047, 2048, 2049, 4097, 100000]:
        for n in (200, 5003, 11008):
            for exact in (False, True):
                _tile(choice, m, n, 32, exact)
        for rows in (64, 128, 256):
            _tile(choice, m, 2048, 32, rows=rows, cols=256)
            _tile(choice, m, 2048, 32, exact=True, rows=rows, cols=256, splits=2)
    # 11008 channels: 43 tiles; 2048 rows as 8 x 256 or 16 x 128 leave the second or third round of tiles a third full
    assert _tile(choice, 2048, 11008, 32)[:2] == (256, 256)


def _greedy(jobs, us, cus):
    """The same by handing out the workgroups of one XCD one after the other."""
    free = [0.0] * (cus // 8)
    heapq.heapify(free)
    for n, t in zip(jobs, us):
        for _ in range(-(-n // 8)):
            heapq.heappush(free, heapq.heappop(free) + t)
    return max(free)


def test_makespan(choice):
    rng = random.Random(4)
    for _ in range(2000):
        jobs = [rng.randint(0, 3000) if rng.random() < 0.7 else 0 for _ in range(3)]
        us = sorted((rng.uniform(5, 100) for _ in range(3)), reverse=True)
        got, want = choice.span(*jobs, *us, 256), _greedy(jobs, us, 256)
        assert abs(got - want) < 1e-6 * max(1.0, want), (jobs, us, got, want)


def test_forms_that_are_asked_for(choice):
    for exact in (False, True):
        for rows in (16, 64, 128, 256):
            for cols in (0, 64, 128, 256):
                for splits in (0, 1, 3):
                    got = _tile(choice, 70, 700, 9, exact, rows, cols, splits)
                    assert got[0] == (min(rows, 128) if exact else rows)
                    if rows == 64 and cols:
                        assert got[1] == cols
                    if rows > 16 and splits:
                        assert got[2] == (3 if splits == 3 else 0)
    assert _tile(choice, 70, 700, 2, rows=64, splits=16)[2] == 1


def test_measured_sides(choice):
    """Where the timings beside the rules are clear."""
    assert _tile(choice, 1, 4096, 86)[:2] == (16, 16)
    assert _tile(choice, 1, 14336, 32)[:2] == (16, 32)
    assert _tile(choice, 48, 14336, 32) == (64, 64, 0)
    assert _tile(choice, 333, 5003, 40)[:2] == (64, 128)
    rows, cols, per = _tile(choice, 64, 4096, 86)
    assert rows == 64 and per
    assert _tile(choice, 4096, 14336, 32)[0] == 256 and _tile(choice, 4096, 14336, 32, exact=True)[0] == 128
    assert choice.direct(8, 64, 4096, 1408) and choice.direct(24, 64, 4096, 1408) and not choice.direct(64, 64, 4096, 1408)
    assert choice.direct(64, 128, 1024, 512) and not choice.direct(128, 128, 1024, 512)
    assert choice.rows(320, 64, 4096, 1408, 0, 0) == 64 and choice.rows(32768, 64, 4096, 1408, 0, 0) == 256
    assert choice.rows(32768, 64, 4096, 1408, 1, 0) == 128
