"""What the choice of a block-scaled product's form costs the caller (CPU: the header is compiled for the host and timed)."""

import ctypes as C
import subprocess
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "pypto_amd" / "csrc"

_SOURCE = """
#include <chrono>
#include "launch_choice.h"
template <typename F>
double best_of(F f) {
  double best = 1e9;
  for (int i = 0; i < 200; ++i) {
    const auto from = std::chrono::steady_clock::now();
    f();
    best = std::min(best, std::chrono::duration<double>(std::chrono::steady_clock::now() - from).count());
  }
  return best;
}
extern "C" double choice(int64_t m, int64_t n, int64_t kb, int exact) {
  return best_of([&] {
    const pto_hip::BlockTile t = pto_hip::choose_block_tile(m, n, kb, exact != 0, 256, 0, 0, 0);
    asm volatile("" ::"r"(&t) : "memory");
  });
}
extern "C" double chain(int count) {  // of dependent multiplications and additions
  return best_of([&] {
    double x = 1.0;
    for (int i = 0; i < count; ++i) {
      x = x * 0.999 + 0.5;
      asm volatile("" : "+m"(x));
    }
  });
}
"""


def test_the_choice_takes_a_few_microseconds_at_any_size(tmp_path):
    """In chains of 600 steps through memory, a microsecond or two, so that a slow machine does not matter.  Many rows, few channels
    and a long k have the most candidates; many rows and many channels the longest schedules."""
    (tmp_path / "time.cpp").write_text(_SOURCE)
    so = tmp_path / "time.so"
    subprocess.run(["g++", "-std=c++17", "-O3", "-shared", "-fPIC", f"-I{CSRC}", str(tmp_path / "time.cpp"), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.choice.argtypes, lib.choice.restype = [C.c_int64] * 3 + [C.c_int], C.c_double
    lib.chain.argtypes, lib.chain.restype = [C.c_int], C.c_double
    unit = lib.chain(600)
    for m, n, kb in ((27035, 244201, 294), (3471, 233773, 2), (4769, 1, 290), (1933, 574, 499), (4001, 134, 101), (4096, 64, 128), (2048, 11008, 32)):
        for exact in (0, 1):
            took = lib.choice(m, n, kb, exact)
            assert took < 4 * unit, (m, n, kb, exact, took / unit)
