"""Tokens of a pass of the experts' FFN (CPU: the header is compiled for the host and called)."""

import ctypes as C
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "pypto_amd" / "csrc"

_SOURCE = """
#include "launch_choice.h"
extern "C" int64_t pass_tokens(int64_t tokens, int64_t top_k, int64_t hidden, int64_t inter, int64_t y_bytes) {
  return pto_hip::expert_pass_tokens(tokens, top_k, hidden, inter, y_bytes);
}
"""


@pytest.fixture(scope="module")
def pass_tokens(tmp_path_factory):
    d = tmp_path_factory.mktemp("pass")
    (d / "pass.cpp").write_text(_SOURCE)
    so = d / "pass.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(d / "pass.cpp"), "-o", str(so)], check=True)
    fn = C.CDLL(str(so)).pass_tokens
    fn.argtypes, fn.restype = [C.c_int64] * 5, C.c_int64
    return fn


def test_the_scratch_of_a_pass_is_bounded(pass_tokens):
    for top_k in (1, 3, 8, 64):
        for hidden in (128, 4096, 16384, 65536):
            for inter in (128, 2048, 65536):
                for y_bytes in (2, 4):
                    for tokens in (1, 7, 600, 1 << 20):
                        n = pass_tokens(tokens, top_k, hidden, inter, y_bytes)
                        assert 1 <= n <= tokens and n * top_k <= 32768
                        assert n * top_k * (hidden * y_bytes + inter) <= 2 << 30


def test_ordinary_layers_keep_the_plan_s_slots(pass_tokens):
    assert pass_tokens(1 << 20, 8, 4096, 1408, 2) == 4096 and pass_tokens(1 << 20, 8, 7168, 2048, 4) == 4096
    assert pass_tokens(1 << 20, 8, 8192, 8192, 4) == 4096 and pass_tokens(2048, 8, 4096, 1408, 2) == 2048
    assert pass_tokens(1 << 20, 64, 65536, 65536, 4) == (2 << 30) // (4 + 65536 + 2048 + 4 * 65536 + 2048) // 64
