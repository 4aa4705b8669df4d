"""The long-context serving operators where timing, scales, probabilities or
bounds lie far apart."""
import numpy as np
import pytest

import longctx_ref as ref
from test_gpu_longctx import Setup, _half_step, _np, _starts, _torch, _type

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(pkg):
    with pkg.Context(num_layers=1, kv_capacity=8) as c:
        yield c


# ------------------------------------------------------------------ timing

@pytest.mark.parametrize("first", ["near", "far"])
def test_prompt_rows_that_arrive_late(pkg, ctx, first):
    """Rows of one row tile out of the L2 while the other's are in it, loaded element by element: the
    result does not depend on which tile comes first."""
    torch = _torch()
    s = Setup(pkg, [2000], 1, 128, 64, "int8", 3)
    away = 1 << 30  # elements between the two tokens, whose 128 heads are a row tile each
    wide = torch.empty(away + 128 * 128 + 1, device="cuda", dtype=torch.bfloat16)
    q = wide[1:].as_strided((2, 128, 128), (away, 128, 1), 1)
    q.copy_(torch.randn(2, 128, 128, generator=torch.Generator().manual_seed(5)).cuda())
    args = (s.dev([0, 2]), s.dev([2000]), s.dev(s.table), 2, 2000)
    want = ctx.kv8_attention(s.cache, q.contiguous(), *args)
    flush = torch.empty(1 << 28, device="cuda", dtype=torch.uint8)
    for i in range(20):
        flush.fill_(i)
        q[0 if first == "near" else 1].float().sum()
        got = torch.full((2, 128, 128), 7.0, device="cuda").bfloat16()
        ctx.kv8_attention(s.cache, q, *args, out=got)
        assert torch.equal(got, want)
    ctx.ops_check()
