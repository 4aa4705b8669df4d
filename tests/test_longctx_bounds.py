"""Bounds near 2^31 of the long-context operators, on the CPU: the arithmetic
that the append kernel's addresses come from (csrc/i4d_seq.h)."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TOP = 2 ** 31 - 1
MOST = 2 ** 30  # tokens of one sequence

SOURCE = """
#include "i4d_seq.h"
extern "C" {
int touched_blocks(int max_q, int tokens, int bs) { return i4d_ops::touched_blocks(max_q, tokens, bs); }
int touched_block(int first, int len, int bs, int j) { return i4d_ops::touched_block(first, len, bs, j); }
}
"""


@pytest.fixture(scope="module")
def seq(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("seq")
    (tmp / "seq.cpp").write_text(SOURCE)
    # an overflow ends the call
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-ftrapv", "-I", os.path.join(ROOT, "4pe_u250_b200", "csrc"),
                    str(tmp / "seq.cpp"), "-o", str(tmp / "seq.so")], check=True)
    return ctypes.CDLL(str(tmp / "seq.so"))


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
def test_blocks_touched_by_any_bound(seq, bs):
    """Enough for every place that the new tokens can have, and no more than one block above what they fill."""
    values = [0, 1, 2, bs - 1, bs, bs + 1, 1000, MOST - 1, MOST, MOST + 1, TOP - bs, TOP - 15, TOP - 1, TOP]
    for max_q in values:
        for tokens in values:
            n = min(max_q, tokens, MOST)
            got = seq.touched_blocks(max_q, tokens, bs)
            want = max(((at + n - 1) // bs - at // bs + 1 for at in range(bs)), default=0) if n else 0
            assert got == want, (max_q, tokens)


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
def test_a_block_lies_in_the_sequence_or_nowhere(seq, bs):
    lengths = [0, 1, bs - 1, bs, bs + 1, 5 * bs + 3, MOST - bs - 1, MOST - 1, MOST]
    most = seq.touched_blocks(TOP, TOP, bs)
    for length in lengths:
        for first in [x for x in lengths if x <= length]:
            for j in [0, 1, 2, 5, 6, most // 2, most - 2, most - 1]:
                at = first // bs + j
                want = at if first < length and at * bs < length else -1
                assert seq.touched_block(first, length, bs, j) == want, (first, length, j)


from test_longctx_refusals import ERR_ARG, ERR_CUDA, _call, _evict, lib  # noqa: E402,F401


@pytest.mark.parametrize("budget,accepted", [(MOST, True), (MOST + 1, False), (TOP - 4095, False), (TOP, False)])
def test_budgets_beyond_any_sequence_are_refused(lib, budget, accepted):  # noqa: F811
    """An index that steps through keep's entries of one row stays in 32 bits."""
    args = _evict(budget=budget, recent=0, keep=0x70000000000)
    assert _call(lib, "i4d_kv8_evict", args) == (ERR_CUDA if accepted else ERR_ARG)
    assert accepted or b"budget" in lib.stub_message()
