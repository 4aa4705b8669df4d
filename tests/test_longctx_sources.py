"""What the overlapped launches of the long-context operators rest on, read from
their sources: every kernel waits first of all for what its stream holds before
it, and loads nothing by the read-only path, whose memory has to be constant
for the kernel's lifetime and whose loads, like those of the cache-hint
intrinsics, the compiler may move ahead of that wait or of a barrier."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "4pe_u250_b200", "csrc")
FILES = ["i4d_ops_common.cuh", "i4d_rope.cuh", "i4d_kv8_cache.cuh", "i4d_kv8_attn.cuh", "i4d_kv8_prompt.cuh", "i4d_logits.cuh"]


def _code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", FILES)
def test_no_load_may_pass_the_wait(name):
    assert not re.findall(r"__ld(?:g|ca|cg|cs|cv|lu)\b|\.nc\b|__restrict__", _code(name))


@pytest.mark.parametrize("name", FILES[1:])
def test_every_kernel_waits_first(name):
    kernels = re.findall(r"__global__[^{;]*?\b(k_\w+)\s*\([^{;]*\)\s*\{\s*(\w+\(\);)", _code(name))
    assert kernels and len(kernels) == _code(name).count("__global__")
    assert all(first == "op_begin();" for _, first in kernels), kernels
