"""The places of a decode batch are counted in 64 bits (attn_plan.h, compiled for the host)."""
import ctypes
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fuel_b200", "csrc")
_SRC = """
#include "attn_plan.h"
extern "C" long long seq_units(const int* lens, int from, int to, int pages, int shift, int tile) {
  return fq::seq_units(lens, from, to, pages, shift, tile);
}
"""


def test_long_sequences_that_share_their_pages(tmp_path):
    (tmp_path / "plan.cpp").write_text(_SRC)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC",
                    "-I", CSRC, "-o", str(tmp_path / "plan.so"), str(tmp_path / "plan.cpp")], check=True)
    units = ctypes.CDLL(str(tmp_path / "plan.so")).seq_units
    units.restype = ctypes.c_longlong
    lens = (ctypes.c_int * 103)(*([2 ** 31 - 1] * 100), 0, -4, 65)
    each = 2 ** 25 + 2                                      # tiles of 64 keys, and the item's own places
    assert units(lens, 0, 100, 2 ** 21, 10, 64) == 100 * each > 2 ** 31
    assert units(lens, 98, 103, 2 ** 21, 10, 64) == 2 * each + 0 + 0 + (2 + 2)
    assert units(lens, 5, 5, 2 ** 21, 10, 64) == 0
    assert units(lens, 102, 103, 1, 5, 64) == 1 + 2         # longer than its row of the page table: that row's 32 keys
