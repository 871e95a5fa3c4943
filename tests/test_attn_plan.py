"""How the attention kernels deal out their work: the index arithmetic of attn_plan.h, compiled for the host."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fuel_b200", "csrc")
_SRC = """
#include "attn_plan.h"
extern "C" {
long long split_begin(long long total, int blocks, int b) { return fq::split_begin(total, blocks, b); }
int split_block(long long total, int blocks, long long tile) { return fq::split_block(total, blocks, tile); }
int split_slot(long long total, int blocks, int b, long long first) { return fq::split_slot(total, blocks, b, first); }
int seq_keys(int len, int max_pages, int shift) { return fq::seq_keys(len, max_pages, shift); }
struct Block { long long first; int len, row; };
void prompt_block(const int* cu, int n, long long rows, long long slot, int size, Block* out) {
  const fq::PromptBlock b = fq::prompt_block(cu, n, rows, slot, size);
  out->first = b.first, out->len = b.len, out->row = b.row;
}
long long prompt_slots(long long rows, int n, int size) { return fq::prompt_slots(rows, n, size); }
int item_units(int tiles) { return fq::item_units(tiles); }
int seq_tiles(int len, int max_pages, int shift, int tile) { return fq::seq_tiles(len, max_pages, shift, tile); }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(_SRC)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC",
                    "-I", CSRC, "-o", str(d / "plan.so"), str(d / "plan.cpp")], check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))
    lib.split_begin.restype = ctypes.c_longlong
    lib.split_begin.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int]
    lib.split_block.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_longlong]
    lib.split_slot.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int, ctypes.c_longlong]
    lib.prompt_block.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_longlong, ctypes.c_int, ctypes.c_void_p]
    lib.prompt_slots.restype = ctypes.c_longlong
    lib.prompt_slots.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int]
    return lib


class _Block(ctypes.Structure):
    _fields_ = [("first", ctypes.c_longlong), ("len", ctypes.c_int), ("row", ctypes.c_int)]


def _blocks(plan, cu, rows, size):
    arr, out = (ctypes.c_int * len(cu))(*cu), []
    for slot in range(plan.prompt_slots(rows, len(cu) - 1, size)):
        b = _Block()
        plan.prompt_block(arr, len(cu) - 1, rows, slot, size, ctypes.byref(b))
        out.append((b.first, b.len, b.row))
    return out


def test_slots_hold_every_block_of_every_prompt_once(plan):
    rng = random.Random(5)
    for _ in range(400):
        lens = [rng.choice((0, rng.randint(0, 4), 128 * rng.randint(0, 6), rng.randint(0, 2000))) for _ in range(rng.randint(1, 9))]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        for size in (128, 256):
            got = _blocks(plan, cu, cu[-1] + rng.choice((0, 1, 300)), size)
            full = [(f, r) for f, n, r in got if r < n]
            assert len(full) == len(set(full)) == sum(-(-n // size) for n in lens)
            for f in {f for f, _ in full}:                      # the longest block of a prompt first
                rows = [r for g, r in full if g == f]
                assert rows == sorted(rows, reverse=True) and rows[-1] == 0 and all(r % size == 0 for r in rows)


def test_boundaries_that_are_none_are_seen(plan):
    for cu in ([0, 20, 40, 90], [0, 20, 40, 30], [0, 20, 40, -3], [0, 20, 40, 2 ** 31 - 1]):
        got = _blocks(plan, cu, 64, 256)
        assert any(n == -1 for _, n, _ in got), cu
        assert {(f, n) for f, n, r in got if n > 0 and r < n} == {(0, 20), (20, 20)}, cu
    assert all(n == -1 for _, n, _ in _blocks(plan, [-5, 70], 64, 128))


def test_runs_cover_the_tiles_and_know_their_block(plan):
    for total in (1, 2, 7, 295, 296, 297, 1000, 4097):
        for blocks in {1, 2, min(total, 296), min(total, 5)}:
            if blocks > total:
                continue
            edges = [plan.split_begin(total, blocks, b) for b in range(blocks + 1)]
            assert edges[0] == 0 and edges[-1] == total
            sizes = [b - a for a, b in zip(edges, edges[1:])]
            assert min(sizes) >= 1 and max(sizes) - min(sizes) <= 1
            for b in range(blocks):
                for t in range(edges[b], edges[b + 1]):
                    assert plan.split_block(total, blocks, t) == b
    total, blocks = 10 ** 12 + 7, 296       # far beyond 32 bits
    for b in (0, 1, 150, 295):
        assert plan.split_block(total, blocks, plan.split_begin(total, blocks, b)) == b
        assert plan.split_block(total, blocks, plan.split_begin(total, blocks, b + 1) - 1) == b


def test_lengths(plan):
    assert [plan.seq_keys(n, 4, 4) for n in (-5, 0, 1, 64, 65, 2 ** 31 - 1)] == [0, 0, 1, 64, 64, 64]
    assert plan.seq_keys(100, 0, 4) == 0
    assert plan.seq_keys(2 ** 31 - 1, 2 ** 31 - 1, 10) == 2 ** 31 - 1
    assert [plan.seq_tiles(n, 1000, 0, 64) for n in (0, 1, 64, 65, 1000, 1001)] == [0, 1, 1, 2, 16, 16]
    assert plan.seq_tiles(2 ** 31 - 1, 2 ** 21, 10, 64) == 2 ** 25


def test_every_piece_has_a_slot_of_its_own_and_is_joined_once(plan):
    """The kernels' walk in Python: each block over its run, then the join of every block's last item if it began there."""
    rng = random.Random(3)
    for _ in range(300):
        lens = [rng.choice((0, 1, 3, 20, 200)) for _ in range(rng.randint(1, 12))]
        items = rng.randint(1, 5)
        spans, at = [], 0
        for n in lens:
            for _ in range(items if n else 0):
                spans.append((at, at + n))
                at += plan.item_units(n)
        total = at
        if not total:
            continue
        assert plan.item_units(0) == 0 and plan.item_units(5) > 5
        blocks = min(total, rng.choice((1, 2, 3, 8, 40)))
        whole, slots, meta = set(), {}, {}
        for b in range(blocks):
            x0, x1 = plan.split_begin(total, blocks, b), plan.split_begin(total, blocks, b + 1)
            for k, (i0, i1) in enumerate(spans):
                a, z = max(i0, x0), min(i1, x1)
                if a >= z:
                    continue
                done = z == i1
                if done and i0 >= x0:
                    whole.add(k)
                else:
                    slot = plan.split_slot(total, blocks, b, i0)
                    assert slot not in slots and slot // 2 == b
                    slots[slot] = (k, a, z)
                    if not done and i0 >= x0:
                        meta[b] = k
        joined = set()
        for b, k in meta.items():
            i0, i1 = spans[k]
            last = plan.split_block(total, blocks, i1 - 1)
            got = [slots[plan.split_slot(total, blocks, b, i0)]] + [slots[2 * c] for c in range(b + 1, last + 1)]
            assert [g[0] for g in got] == [k] * len(got)
            assert [g[1] for g in got] == [i0] + [g[2] for g in got[:-1]] and got[-1][2] == i1
            joined.add(k)
        assert joined | whole == set(range(len(spans))) and not joined & whole
