"""The long-context serving operators where timing, scales, probabilities or
bounds lie far apart."""
import numpy as np
import pytest

import longctx_ref as ref
from test_gpu_longctx import Setup, _np, _run_attention, _torch, _type

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


# ----------------------------------------------------------- probabilities

def _attend(pkg, ctx, s, q, n, length, scale, floor=0.0, one_part=2.0 ** -11):
    """Output within the bounds of tests/test_gpu_longctx.py (`one_part`: the probabilities' rounding for 16-bit outputs), and
    `floor` of a row's greatest weight for each token that it sees.  The greatest weight is at most 1 times the
    greatest value scale, and a token's code at most its |v| over its own scale."""
    torch = _torch()
    lse = torch.empty(n, q.shape[1], device="cuda")
    out = ctx.kv8_attention(s.cache, q, s.dev([0, n]), s.dev([length]), s.dev(s.table), n, length, scale=scale, lse=lse)
    ctx.ops_check()
    w_out, w_lse, _, mag, size = ref.attention(s.ref(), _np(q), [0, n], [length], s.table, scale)
    dx = size * ((s.dim / 16 + 6) * 2.0 ** -23 + 2.0 ** -22) + 2.0 ** -21
    p = 2 * dx + (2.0 ** -21 if q.dtype == torch.float32 else one_part) + length / 16 * 2.0 ** -23
    err = mag * p[..., None]
    if floor:
        c = s.ref()
        blocks = s.table[0, :-(-length // s.bs)]
        codes = np.abs(c.codes[1][blocks]).transpose(1, 0, 2, 3).reshape(s.heads, -1, s.dim)[:, :length].sum(1)
        err = err + floor * np.repeat(codes * c.scale[1][blocks].max(0)[:, None], q.shape[1] // s.heads, 0)
    # (FP16 values under 2^-14 lie 2^-24 apart)
    assert np.all(np.abs(_np(out) - w_out) <= err + _half(q.dtype) * (np.abs(w_out) + err) + (2.0 ** -25 if q.dtype == torch.float16 else 1e-30))
    assert np.all(np.abs(_np(lse) - w_lse) <= dx + length / 16 * 2.0 ** -23 + 2.0 ** -22 * (np.abs(w_lse) + 1))
    return out


def _half(t):
    return _torch().finfo(t).eps / 2


def _sink(pkg, kind, length, at, seed):
    """Equal scores, but for one token at `at` of value 0; positive values, so that errors of equal probabilities add up."""
    torch = _torch()
    s = Setup(pkg, [length], 1, 64, 64, kind, seed)
    top = 12 if kind == "int8" else 10
    v = torch.from_numpy(s.rng.integers(6, top, s.cache.v.shape) * (8.0 if kind == "int8" else 16.0)).cuda()
    s.cache.k.zero_()
    s.cache.v.copy_(v.to(s.cache.v.dtype))
    for x in (s.cache.k_scale, s.cache.v_scale):
        x.fill_(1.0)
    block, slot = int(s.table[0, at // 64]), at % 64
    s.cache.k[block, 0, slot, 0] = 64
    s.cache.v[block, 0, slot] = 0
    return s


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kind,at", [("int8", 0), ("e4m3", 0), ("int8", 20001), ("e4m3", 32768)])
@pytest.mark.parametrize("down", [22.3, 26.7, 60.2])
def test_small_probabilities_of_a_long_tail(pkg, ctx, name, kind, at, down):
    """32768 tokens of 2^-down of the greatest weight, whose own value is 0: their relative precision is the output's.  Ones
    under FP16's range for 16-bit outputs too, though those of FP16 are then 0."""
    torch = _torch()
    s = _sink(pkg, kind, 32769, at, 83)
    q = torch.zeros(1, 3, 64, device="cuda", dtype=_type(name))
    q[:, :, 0] = 1
    _attend(pkg, ctx, s, q, 1, 32769, down * np.log(2) / 64)


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_far_scores_of_many_draws(pkg, ctx, name, kind):
    """Where a row's greatest weight meets a code of 0, what is left is the next token's, however small."""
    torch = _torch()
    for seed in range(20):
        s = Setup(pkg, [300], 2, 128, 32, kind, 100 + seed)
        q = torch.randn(1, 8, 128, generator=torch.Generator().manual_seed(seed)).to(_type(name)).cuda()
        _attend(pkg, ctx, s, q, 1, 300, 0.2 * (1 + seed % 5))
