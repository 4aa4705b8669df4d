"""The order of copies and waits in a warp's ring (csrc/i4d_ring.h), on the
CPU, with barriers whose phases end when the test says so."""
import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "i4d_ring.h"
using namespace i4d_ops;
namespace {
struct Event { int kind, slot, item; };  // 0 copy, 1 wait (item: parity), 2 use, 3 free
template <int SLOTS>
int simulate(const int* tables, int n_tables, int first, int step, int late, Event* out) {
    Ring ring;
    int n = 0, waits = 0;
    for (int t = 0; t < n_tables; ++t) {
        auto issue = [&](int item, int slot) {
            if (item < tables[t]) out[n++] = {0, slot, item};
        };
        auto wait = [&](int slot, uint32_t parity) { out[n++] = {1, slot, static_cast<int>(parity)}; return ++waits != late; };
        ring_fill<SLOTS>(ring, first, step, issue);
        ring_walk<SLOTS>(ring, first, step, tables[t], issue, wait, [&] { out[n++] = {3, 0, 0}; }, [&](int item, int slot, bool landed) {
            if (landed) out[n++] = {2, slot, item};
            return landed;
        });
    }
    return n;
}
}
extern "C" int run(int slots, const int* tables, int n_tables, int first, int step, int late, Event* out) {
    return slots == 3 ? simulate<3>(tables, n_tables, first, step, late, out) : simulate<6>(tables, n_tables, first, step, late, out);
}
"""


class Event(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int), ("slot", ctypes.c_int), ("item", ctypes.c_int)]


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("ring")
    (tmp / "ring.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "4pe_u250_b200", "csrc"), str(tmp / "ring.cpp"),
                    "-o", str(tmp / "ring.so")], check=True)
    lib = ctypes.CDLL(str(tmp / "ring.so"))

    def call(slots, tables, first, step, late):
        out = (Event * (4 * sum(tables) + 100))()
        n = lib.run(slots, (ctypes.c_int * len(tables))(*tables), len(tables), first, step, late, out)
        return [(e.kind, e.slot, e.item) for e in out[:n]]
    return call


def _check(events, slots, tables, first, step, late):
    copies, done = [0] * slots, [0] * slots  # copies started into a slot, and phases of its barrier waited for
    holds = [None] * slots                   # item that a slot's copy in flight or landed brings
    waits, gave_up, used = 0, None, []
    for at, (kind, slot, item) in enumerate(events):
        if kind == 0:
            assert gave_up is None, "a copy after a wait that gave up"
            assert copies[slot] == done[slot] and holds[slot] is None, "a copy into a slot that is not free"
            copies[slot] += 1
            holds[slot] = item
        elif kind == 1:
            waits += 1
            assert copies[slot] == done[slot] + 1 or gave_up is not None, "a wait for no copy"
            # the phase that the copy in flight ends is number copies - 1: its parity
            assert item == (copies[slot] - 1) % 2, "a wait for another phase's parity"
            if gave_up is None and waits == late:
                gave_up = at
            elif gave_up is None:
                done[slot] += 1
            else:
                done[slot] = copies[slot]
        elif kind == 2:
            assert gave_up is None and holds[slot] == item
            holds[slot] = None
            used.append(item)
    if gave_up is None:
        assert used == [i for n in tables for i in range(first, n, step)]
    assert done == copies, "a copy that nothing waited for"


@pytest.mark.parametrize("slots", [3, 6])
@pytest.mark.parametrize("first", [0, 3])
def test_ring_waits_for_every_copy_once(run, slots, first):
    rng = random.Random(slots * 10 + first)
    for _ in range(60):
        tables = [rng.choice([0, 1, 3, 4, 5, 12, 33, 256, 257]) for _ in range(rng.randint(1, 4))]
        _check(run(slots, tables, first, 4, 0), slots, tables, first, 4, 0)


@pytest.mark.parametrize("slots", [3, 6])
def test_ring_after_a_wait_that_gave_up(run, slots):
    """No copy and no use after it, in later tables neither, and a wait by the right parity for each copy in flight."""
    rng = random.Random(slots)
    for _ in range(200):
        tables = [rng.choice([1, 3, 4, 5, 12, 33, 130]) for _ in range(rng.randint(1, 4))]
        items = sum(-(-n // 4) for n in tables)
        late = rng.randint(1, items)
        _check(run(slots, tables, 0, 4, late), slots, tables, 0, 4, late)
