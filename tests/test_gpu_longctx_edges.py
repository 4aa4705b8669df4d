"""The long-context serving operators where timing, scales, probabilities or
bounds lie far apart."""
import numpy as np
import pytest

from test_gpu_longctx import Setup, _np, _run_attention, _torch

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


# ------------------------------------------------------------------ scales

@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("group", [1, 4])
def test_zero_values_before_large_ones(pkg, ctx, name, kind, group):
    """The first rows see only a block of zeros, whose scale is 2^-126, in tiles whose later blocks have scales of 8 and more."""
    torch = _torch()
    g = torch.Generator().manual_seed(7)
    s = Setup(pkg, [40], 2, 64, 16, kind, 73)
    k, v = torch.randn(40, 2, 64, generator=g), torch.randn(40, 2, 64, generator=g) * 1000
    v[:16] = 0
    ctx.kv8_append(s.cache, k.cuda(), v.cuda(), s.dev([0, 40]), s.dev([40]), s.dev(s.table), 40)
    assert s.cache.v_scale[s.table[0, 0]].max() == 2.0 ** -126 and s.cache.v_scale[s.table[0, 1]].min() >= 4
    for n in (40, 35):  # (row tiles that end at the block's border, and that do not)
        _, out = _run_attention(pkg, ctx, s, [n], [40], 2 * group, name, 0)
        assert torch.all(out[:16 - 40 + n] == 0)


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("group", [1, 4])
@pytest.mark.parametrize("up", [1, 2 ** 7])
def test_value_scales_of_exactly_zero(pkg, ctx, name, group, up):
    """A scale of 0 makes zeros of its block's codes, however far its scores lie above or below the others'."""
    s = Setup(pkg, [60], 2, 64, 16, "int8", 79)
    for block in s.table[0, [0, 2]]:
        s.cache.v_scale[int(block)] = 0
        s.cache.k_scale[int(block)] *= up
    for n, window in ((60, 0), (55, 0), (55, 9)):
        _run_attention(pkg, ctx, s, [n], [60], 2 * group, name, window)
    s.cache.v_scale.zero_()
    _, out = _run_attention(pkg, ctx, s, [60], [60], 2 * group, name, 0)
    assert np.all(_np(out) == 0)
