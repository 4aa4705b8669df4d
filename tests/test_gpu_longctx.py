"""The long-context serving operators on the GPU against their 64-bit
definitions (tests/longctx_ref.py)."""
import itertools

import numpy as np
import pytest

import longctx_ref as ref

pytestmark = pytest.mark.gpu

NAMES = ("f32", "bf16", "f16")


def _torch():
    import torch
    return torch


def _type(name):
    torch = _torch()
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _half_step(t):
    return _torch().finfo(t).eps / 2


def _np(x):
    return x.detach().double().cpu().numpy()


@pytest.fixture(scope="module")
def ctx(pkg):
    with pkg.Context(num_layers=1, kv_capacity=8) as c:
        yield c


# ------------------------------------------------------------------- rope

def _rope_bound(x, y, magnitude, t, interleaved, half):
    """Angle: 2^-24 of an eighth of a turn (4.7e-8) and the table's 2^-34; sine
    and cosine 2 units of 2^-24 each, magnitude and three FP32 roundings of the
    pair's products; then half a step of the output type."""
    a = np.abs(x)
    pair = a.copy()
    if interleaved:
        pair[..., 0:2 * half:2] = a[..., 0:2 * half:2] + a[..., 1:2 * half:2]
        pair[..., 1:2 * half:2] = pair[..., 0:2 * half:2]
    else:
        pair[..., :half] = a[..., :half] + a[..., half:2 * half]
        pair[..., half:2 * half] = pair[..., :half]
    err = pair * magnitude * (4.7e-8 + 1e-9 + 6 * 2.0 ** -24)
    return err + _half_step(t) * (np.abs(y) + err) + 1e-30


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,scaling", [
    (1, 1, 1, 64, 64, "none"), (3, 5, 2, 96, 32, "parts"), (33, 4, 4, 80, 80, "base"), (7, 32, 8, 128, 128, "linear"),
    (2, 3, 1, 256, 256, "none"), (5, 2, 2, 20, 6, "none"), (4, 2, 1, 18, 18, "parts"),
    (2401, 3, 1, 64, 32, "none"), (2401, 2, 1, 20, 6, "none"), (2401, 1, 2, 256, 256, "base")])
def test_rope(pkg, ctx, name, interleaved, tokens, heads, kv, dim, rot, scaling):
    torch = _torch()
    t = _type(name)
    g = torch.Generator().manual_seed(tokens * 100 + dim)
    q = torch.randn(tokens, heads, dim, generator=g).to(t).cuda()
    k = torch.randn(tokens, kv, dim, generator=g).to(t).cuda()
    pos = torch.randint(-5000, 2 ** 31 - 1, (tokens,), generator=g, dtype=torch.int64).int()
    pos[0] = 0
    factor = 1.0 if scaling == "none" else 8.0
    table = pkg.RopeTable(rot, scaling=scaling, factor=factor, magnitude=1.25)
    f = ref.frequencies(rot, scaling=scaling, factor=factor)
    # a 64-bit angle of a far position is itself off by 2^-53 of the angle
    far = np.abs(pos.numpy()).max() * 2.0 ** -52
    for inverse in (False, True):
        qo, ko = ctx.rope(q, k, pos.cuda(), table, interleaved=interleaved, inverse=inverse)
        for x, y in ((q, qo), (k, ko)):
            want = ref.rope(_np(x), pos.numpy(), f, 1.25, interleaved, inverse)
            bound = _rope_bound(_np(x), want, 1.25, t, interleaved, rot // 2)
            assert np.all(np.abs(_np(y) - want) <= bound + far * 2.5 * np.abs(_np(x)).max())
            assert torch.equal(y[..., rot:], x[..., rot:])


def test_rope_strided_in_place_and_without_k(pkg, ctx):
    torch = _torch()
    qkv = torch.randn(9, 3 * 4 * 64, device="cuda").bfloat16()
    q, k = qkv.view(9, 12, 64)[:, :4], qkv.view(9, 12, 64)[:, 4:8]
    pos = torch.arange(9, device="cuda", dtype=torch.int32) * 1000
    table = pkg.RopeTable(64)
    want = ctx.rope(q.contiguous(), k.contiguous(), pos, table)
    alone, none = ctx.rope(q, None, pos, table)
    assert none is None and torch.equal(alone, want[0])
    v = qkv[:, 8 * 64:].clone()
    got = ctx.rope(q, k, pos, table, q_out=q, k_out=k)
    assert got[0].data_ptr() == qkv.data_ptr()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 8 * 64:], v)
    # rows of a transposed layout [heads, tokens, dim], and one element off the 16-byte boundary
    flat = torch.randn(1 + 4 * 9 * 64, device="cuda").bfloat16()
    off = flat[1:].view(4, 9, 64).transpose(0, 1)
    got, _ = ctx.rope(off, None, pos, table, interleaved=False)
    want, _ = ctx.rope(off.contiguous(), None, pos, table, interleaved=False)
    assert torch.equal(got, want)


def test_rope_rotates_back(pkg, ctx):
    torch = _torch()
    x = torch.randn(50, 2, 128, device="cuda")
    pos = torch.randint(0, 10 ** 9, (50,), device="cuda", dtype=torch.int32)
    table = pkg.RopeTable(128)
    there, _ = ctx.rope(x, None, pos, table)
    back, _ = ctx.rope(there, None, pos, table, inverse=True)
    # two rotations of a pair of norm r, each off by at most 4.2e-7 (|a| + |b|) <= 6e-7 r
    r = (x[..., 0::2] ** 2 + x[..., 1::2] ** 2).sqrt().repeat_interleave(2, -1)
    assert torch.all((back - x).abs() <= 1.2e-6 * r + 1e-7)


# ------------------------------------------------------------------- cache

class Setup:
    """A pool with a random order of blocks and normal values, on the GPU and in 64 bits."""

    def __init__(self, pkg, lens, heads, dim, bs, kind, seed, spread=3):
        torch = _torch()
        self.rng = np.random.default_rng(seed)
        self.bs, self.heads, self.dim, self.kind, self.lens = bs, heads, dim, kind, list(lens)
        need = [max(1, -(-n // bs)) for n in lens]
        blocks, wide = sum(need) + 2, max(need) + 1
        order = self.rng.permutation(blocks)
        self.table = np.zeros((len(lens), wide), np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.cache = pkg.KV8Cache.empty(blocks, heads, bs, dim, kind)
        low = -6 if kind == "int8" else -8
        for codes, scale in ((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale)):
            scale.copy_(torch.from_numpy(2.0 ** self.rng.integers(low, low + spread, (blocks, heads))))
            x = torch.from_numpy(self.rng.standard_normal((blocks, heads, bs, dim))).cuda() / scale[..., None, None]
            x = x.clamp(-ref.TOP[kind], ref.TOP[kind])
            codes.copy_((x.round() if kind == "int8" else x).to(codes.dtype))

    def ref(self):
        c = self.cache
        return ref.Cache(_np(c.k), _np(c.v), _np(c.k_scale), _np(c.v_scale), self.kind)

    def dev(self, x):
        torch = _torch()
        return torch.as_tensor(np.asarray(x, np.int32)).cuda()


def _starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def _same_cache(cache, want):
    assert np.array_equal(_np(cache.k_scale), want.scale[0]) and np.array_equal(_np(cache.v_scale), want.scale[1])
    assert np.array_equal(_np(cache.k), want.codes[0]) and np.array_equal(_np(cache.v), want.codes[1])


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("bs,dim,heads", [(16, 64, 3), (32, 128, 2), (64, 80, 1), (128, 256, 2), (16, 16, 1)])
def test_append_and_read(pkg, ctx, name, kind, bs, dim, heads):
    torch = _torch()
    q_lens, lens = [1, 0, 3 * bs + 5, bs, 7, 1], [1, bs, 3 * bs + 5, 2 * bs, bs + 3, bs + 1]
    s = Setup(pkg, lens, heads, dim, bs, kind, 7 + bs + dim)
    start = _starts(q_lens)
    new = [s.rng.standard_normal((start[-1], heads, dim)) * np.exp(s.rng.standard_normal((start[-1], heads, 1))) * 4 for _ in range(2)]
    k, v = (torch.from_numpy(x).to(_type(name)).cuda() for x in new)
    if name == "f32":
        k[2, 0, 0], k[3, 0, 1], v[4, 0, 2] = float("nan"), float("inf"), -float("inf")
    if start[-1] > 9:
        v[9] = 0
    want = s.ref()
    want.append((_np(k), _np(v)), start, lens, s.table)
    before = s.cache.k.clone()
    ctx.kv8_append(s.cache, k, v, s.dev(start), s.dev(lens), s.dev(s.table), max(q_lens))
    ctx.ops_check()
    _same_cache(s.cache, want)
    assert not torch.equal(before.view(torch.int8), s.cache.k.view(torch.int8))
    got = ctx.kv8_read(s.cache, s.dev(start), s.dev(lens), s.dev(s.table), max(q_lens), int(start[-1]))
    for which in range(2):
        for b, n in enumerate(q_lens):
            for h in range(heads):
                idx = np.arange(lens[b] - n, lens[b])
                assert np.array_equal(_np(got[which])[start[b]:start[b + 1], h], want.tokens(which, s.table[b], h, idx))


def test_append_token_by_token_is_within_one_step(pkg, ctx):
    """Codes rewritten for rising scales: the sum of the roundings stays under one step of the last scale."""
    torch = _torch()
    s = Setup(pkg, [64], 1, 64, 64, "int8", 3)
    x = torch.randn(64, 1, 64, device="cuda") * torch.exp(torch.linspace(-6, 4, 64, device="cuda"))[:, None, None]
    for i in range(64):
        ctx.kv8_append(s.cache, x[i:i + 1], x[i:i + 1], s.dev([0, 1]), s.dev([i + 1]), s.dev(s.table), 1)
    k, _ = ctx.kv8_read(s.cache, s.dev([0, 64]), s.dev([64]), s.dev(s.table), 64, 64)
    step = s.cache.k_scale[int(s.table[0, 0]), 0]
    assert torch.all((k.float() - x).abs() <= step)


def test_append_strided_rows_leave_the_rest(pkg, ctx):
    torch = _torch()
    s = Setup(pkg, [20, 5], 2, 64, 16, "e4m3", 5)
    qkv = torch.randn(9, 6, 64, device="cuda").half()
    k, v = qkv[:, 2:4], qkv[:, 4:6]
    want = s.ref()
    want.append((_np(k), _np(v)), [0, 4, 6], [20, 5], s.table)
    # three rows behind the last sequence are not read; slots behind the last token keep their bytes
    ctx.kv8_append(s.cache, k, v, s.dev([0, 4, 6]), s.dev([20, 5]), s.dev(s.table), 4)
    _same_cache(s.cache, want)
    out = torch.full((9, 2, 64), 7.0, device="cuda").bfloat16()
    ctx.kv8_read(s.cache, s.dev([0, 4, 6]), s.dev([20, 5]), s.dev(s.table), 4, 9, k_out=out)
    assert torch.all(out[6:] == 7)
    # one element off the 16-byte boundary: the narrow loads
    flat = torch.randn(1 + 6 * 2 * 64, device="cuda").half()
    k2 = flat[1:].view(6, 2, 64)
    want.append((_np(k2), _np(k2)), [0, 4, 6], [20, 5], s.table)
    ctx.kv8_append(s.cache, k2, k2, s.dev([0, 4, 6]), s.dev([20, 5]), s.dev(s.table), 4)
    _same_cache(s.cache, want)


# --------------------------------------------------------------- attention

def _attention_bounds(t, dim, out, mag, size, lse, rows):
    """x = score in nats: FP32 sums of dim products (dim / 16 + 6 roundings of 2^-23 of sum |q k|), the split of an
    FP32 row (2^-22), the exponential (2^-21).  Probabilities: relative 2 dx, and 2^-11 for their FP16 part (2^-21
    where they are in two).  Sums over tokens: FP32, 2^-23 for each of rows / 16 steps."""
    torch = _torch()
    dx = size * ((dim / 16 + 6) * 2.0 ** -23 + 2.0 ** -22) + 2.0 ** -21
    p = 2 * dx + (2.0 ** -21 if t == torch.float32 else 2.0 ** -11) + rows / 16 * 2.0 ** -23
    b_out = mag * p[..., None] + _half_step(t) * (np.abs(out) + mag * p[..., None]) + 1e-30
    fine = np.where(np.isfinite(lse), lse, 0.0)
    return b_out, dx + rows / 16 * 2.0 ** -23 + 2.0 ** -22 * (np.abs(fine) + 1), 2 * dx + 2.0 ** -21 * (1 + np.abs(fine))


def _run_attention(pkg, ctx, s, q_lens, lens, heads, name, window, max_length=None, scale=None, extra=0, seed=0, table=None, bad=None):
    torch = _torch()
    t = _type(name)
    start = _starts(q_lens)
    total = int(start[-1]) + extra
    g = torch.Generator().manual_seed(seed + total)
    q = (torch.randn(total, heads, s.dim, generator=g) * 1.5).to(t).cuda()
    out = torch.full((total, heads, s.dim), 7.0, device="cuda", dtype=t)
    lse = torch.full((total, heads), 7.0, device="cuda")
    max_length = max_length or max(lens)
    weights = torch.rand(len(lens), s.heads, max_length + 3, generator=g).cuda()
    before = weights.clone()
    table = s.table if table is None else table
    ctx.kv8_attention(s.cache, q, s.dev(start), s.dev(lens), s.dev(table), max(q_lens), max_length, scale=scale,
                      window=window, out=out, lse=lse, weights=weights)
    scale = 1 / np.sqrt(s.dim) if scale is None else scale
    w_out, w_lse, sums, mag, size = ref.attention(s.ref(), _np(q), start, lens, table, scale, window)
    n = int(start[-1])
    b_out, b_lse, b_p = _attention_bounds(t, s.dim, w_out, mag, size, w_lse, max(lens))
    assert np.all(np.abs(_np(out) - w_out)[:n] <= b_out[:n])
    got = _np(lse)[:n]
    gone = ~np.isfinite(w_lse[:n])
    assert np.array_equal(got[gone], w_lse[:n][gone])
    assert np.all(np.abs(got[~gone] - w_lse[:n][~gone]) <= b_lse[:n][~gone])
    assert torch.all(out[n:] == 7) and torch.all(lse[n:] == 7)  # rows behind the last sequence
    group = heads // s.heads
    for b, length in enumerate(lens):
        rel = b_p[start[b]:start[b + 1]].max() if q_lens[b] else 0.0
        add = (_np(weights) - _np(before))[b]
        # the FP32 sum: rows of the head, each rounded, and the entry's own rounding
        slack = sums[b] * (rel + 2.0 ** -22) + 2.0 ** -23 * (np.abs(_np(before))[b][:, :length] + sums[b]) + 2.0 ** -24 * q_lens[b] * group * sums[b]
        assert np.all(np.abs(add[:, :length] - sums[b]) <= slack)
        assert np.all(add[:, length:] == 0)
    # without the weights and lse: the same output
    again = ctx.kv8_attention(s.cache, q[:n], s.dev(start), s.dev(lens), s.dev(table), max(q_lens), max_length, scale=scale, window=window)
    assert torch.equal(again, out[:n])
    if bad:  # the host hears of what the device skipped, once
        with pytest.raises(pkg.I4DError, match=bad):
            ctx.ops_check()
    ctx.ops_check()
    return q, out


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("bs,dim,kv,group", [(16, 64, 2, 1), (32, 128, 1, 4), (64, 128, 2, 8), (128, 256, 1, 2), (16, 80, 2, 3),
                                             (64, 96, 1, 16), (32, 16, 2, 2), (64, 192, 1, 7)])
def test_attention_single_tokens(pkg, ctx, name, kind, bs, dim, kv, group):
    lens = [1, 2, 15, 16, 17, 33, 300, 517]
    s = Setup(pkg, lens, kv, dim, bs, kind, bs + dim + group)
    _run_attention(pkg, ctx, s, [1] * len(lens), lens, kv * group, name, 0)
    _run_attention(pkg, ctx, s, [1] * len(lens), lens, kv * group, name, 20, extra=3)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("bs,dim,kv,group", [(16, 64, 2, 2), (64, 128, 1, 4), (128, 128, 2, 1), (32, 256, 1, 2), (32, 112, 1, 8)])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_prompts(pkg, ctx, name, kind, bs, dim, kv, group, window):
    q_lens, lens = [3, 0, 130, 1, 64, 200], [3, 40, 130, 77, 300, 201]
    s = Setup(pkg, lens, kv, dim, bs, kind, bs + dim + 1)
    _run_attention(pkg, ctx, s, q_lens, lens, kv * group, name, window, extra=2)


def test_attention_many_chunks(pkg, ctx):
    """A long context among short ones, split over the token axis; max_length above every length."""
    lens = [5000, 1, 260, 4097]
    for name, kind in (("bf16", "int8"), ("f32", "e4m3")):
        s = Setup(pkg, lens, 2, 128, 32, kind, 11)
        _run_attention(pkg, ctx, s, [1] * 4, lens, 8, name, 0)
        _run_attention(pkg, ctx, s, [1] * 4, lens, 8, name, 1000, max_length=5024)
        _run_attention(pkg, ctx, s, [2, 1, 3, 1], lens, 4, name, 0)


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_attention_scales_far_apart(pkg, ctx, name):
    """Blocks whose value scales differ by 2^40, and zero blocks, cost the others no precision: bounds are relative to sum p |v|."""
    s = Setup(pkg, [200, 40], 2, 64, 16, "int8", 13)
    s.cache.v_scale[::2] *= 2.0 ** 40
    s.cache.k_scale[::2] *= 2.0 ** -9
    s.cache.v[int(s.table[0, 3])] = 0
    s.cache.v_scale[int(s.table[0, 3])] = 2.0 ** -126
    s.cache.k_scale[int(s.table[0, 5])] *= 8
    for window in (0, 17):
        _run_attention(pkg, ctx, s, [1, 30], [200, 40], 4, name, window)


def test_attention_far_scores_and_small_queries(pkg, ctx):
    torch = _torch()
    s = Setup(pkg, [300], 1, 128, 32, "int8", 17)
    for name, size in (("bf16", 1e30), ("bf16", 1e-30), ("f32", 1e-3), ("f32", 30.0), ("f16", 1e-4)):
        t = _type(name)
        q = (torch.randn(1, 1, 128, device="cuda") * size).to(t)
        scale = 3e-30 if size == 1e30 else 1e29 if size == 1e-30 else 1 / np.sqrt(128)
        lse = torch.empty(1, 1, device="cuda")
        out = ctx.kv8_attention(s.cache, q, s.dev([0, 1]), s.dev([300]), s.dev(s.table), 1, 300, scale=scale, lse=lse)
        w_out, w_lse, _, mag, sz = ref.attention(s.ref(), _np(q), [0, 1], [300], s.table, scale)
        b_out, b_lse, _ = _attention_bounds(t, 128, w_out, mag, sz, w_lse, 300)
        assert np.all(np.abs(_np(out) - w_out) <= b_out) and np.all(np.abs(_np(lse) - w_lse) <= b_lse)


def test_attention_nan_rows_and_garbage_behind_the_end(pkg, ctx):
    torch = _torch()
    for group, n in ((2, 3), (2, 100)):
        s = Setup(pkg, [120], 1, 128, 64, "e4m3", 19)
        q = torch.randn(n, group, 128, device="cuda").bfloat16()
        args = (s.dev([0, n]), s.dev([120]), s.dev(s.table), n, 120)
        want = ctx.kv8_attention(s.cache, q, *args)
        # NaN codes in the slots behind the last token, NaN in one row's query
        s.cache.k.view(torch.int8)[int(s.table[0, 1]), :, 120 - 64:] = 0x7f
        s.cache.v.view(torch.int8)[int(s.table[0, 1]), :, 120 - 64:] = 0x7f
        q[1, 1, 5] = float("nan")
        got = ctx.kv8_attention(s.cache, q, *args)
        assert torch.all(torch.isnan(got[1, 1]))
        keep = torch.ones(n, group, dtype=torch.bool, device="cuda")
        keep[1, 1] = False
        assert torch.equal(got[keep], want[keep])


def test_attention_strides(pkg, ctx):
    torch = _torch()
    s = Setup(pkg, [60, 33], 2, 64, 16, "int8", 23)
    for n in (1, 25):
        start, lens, table = s.dev([0, n, 2 * n]), s.dev([60, 33]), s.dev(s.table)
        qkv = torch.randn(2 * n, 8, 64, device="cuda").half()
        want = ctx.kv8_attention(s.cache, qkv[:, :4].contiguous(), start, lens, table, n, 60)
        assert torch.equal(ctx.kv8_attention(s.cache, qkv[:, :4], start, lens, table, n, 60), want)
        turned = torch.empty(4, 2 * n, 64, device="cuda").half().transpose(0, 1)
        ctx.kv8_attention(s.cache, qkv[:, :4], start, lens, table, n, 60, out=turned)
        assert torch.equal(turned, want)
        odd = torch.empty(2 * n, 4, 65, device="cuda").half()[:, :, 1:]
        odd.copy_(qkv[:, :4])
        assert torch.equal(ctx.kv8_attention(s.cache, odd, start, lens, table, n, 60), want)
        same = qkv[:, :1].expand(-1, 4, -1)  # one head's rows for all heads
        assert torch.equal(ctx.kv8_attention(s.cache, same, start, lens, table, n, 60),
                           ctx.kv8_attention(s.cache, same.contiguous(), start, lens, table, n, 60))


# ------------------------------------------------------------------- evict

@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("bs,dim,heads", [(16, 64, 2), (32, 128, 1), (64, 80, 2), (128, 16, 1)])
@pytest.mark.parametrize("budget,recent", [(40, 0), (100, 30), (64, 64), (150, 1), (1, 0)])
def test_evict(pkg, ctx, kind, bs, dim, heads, budget, recent):
    torch = _torch()
    lens = [1, budget, budget + 1, 333, 0, 2100]
    s = Setup(pkg, lens, heads, dim, bs, kind, budget + bs)
    most = max(lens) + 5
    w = s.rng.integers(0, 12, (len(lens), heads, most)).astype(np.float32)  # many ties
    w[3, :, :50] = s.rng.standard_normal((heads, 50))
    for b, n in enumerate(lens):
        w[b, :, n:] = 0
    want = s.ref()
    lens_w, keep_w, w_w = want.evict(s.table, lens, w.astype(np.float64), budget, recent)
    weights = torch.from_numpy(w).cuda()
    lo, keep, left = ctx.kv8_evict(s.cache, s.dev(lens), s.dev(s.table), weights, budget, recent, most - 5)
    ctx.ops_check()
    assert left is weights and lo.tolist() == lens_w and np.array_equal(_np(left), w_w)
    for b, h in itertools.product(range(len(lens)), range(heads)):
        got = keep[b, h].tolist()
        assert got == list(keep_w[b][h]) + [-1] * (budget - len(keep_w[b][h]))
    got_k = _np(s.cache.k)
    for b, n in enumerate(lens_w):  # the kept slots; what lies behind the new length is free
        for j in range(-(-n // bs)):
            part, blk = min(bs, n - j * bs), s.table[b, j]
            assert np.array_equal(got_k[blk, :, :part], want.codes[0][blk, :, :part])
            assert np.array_equal(_np(s.cache.v)[blk, :, :part], want.codes[1][blk, :, :part])
            assert np.array_equal(_np(s.cache.k_scale)[blk], want.scale[0][blk])
            assert np.array_equal(_np(s.cache.v_scale)[blk], want.scale[1][blk])


def test_evict_weights_apart_nan_and_infinities(pkg, ctx):
    torch = _torch()
    s = Setup(pkg, [50], 1, 32, 16, "int8", 29)
    w = torch.zeros(1, 1, 50)
    w[0, 0, 7], w[0, 0, 8], w[0, 0, 9], w[0, 0, 10], w[0, 0, 11] = float("nan"), float("inf"), -float("inf"), -1.0, -0.0
    _, keep, left = ctx.kv8_evict(s.cache, s.dev([50]), s.dev(s.table), w.cuda(), 46, 2, 50, weights_out=torch.full((1, 1, 50), 9.0).cuda())
    # 44 of the first 48: all but NaN, -inf, -1 and, of the equal zeros, the last
    assert keep[0, 0].tolist() == [i for i in range(50) if i not in (7, 9, 10, 47)]
    assert left[0, 0, 46:].tolist() == [0.0] * 4 and left[0, 0, 7].item() == float("inf")


# ------------------------------------------------------------------ logits

@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 33), (2, 4099), (5, 32000), (1, 128001), (300, 517)])
def test_logits(pkg, ctx, name, rows, vocab):
    torch = _torch()
    t = _type(name)
    rng = np.random.default_rng(rows + vocab)
    x = torch.from_numpy(rng.standard_normal((rows, vocab)) * 3).to(t)
    hist = rng.integers(-3, vocab + 3, (rows, 90))
    hist[:, 30:60] = hist[:, :30]
    hlen, plen = rng.integers(0, 91, rows), rng.integers(0, 40, rows)
    ids, vals, blen = rng.integers(-2, vocab + 2, (rows, 45)), rng.standard_normal((rows, 45)).astype(np.float32) * 4, rng.integers(0, 46, rows)
    ids[:, 40:] = ids[:, :1]  # one id several times
    mask = rng.integers(0, 2 ** 32, (rows, -(-vocab // 32)), dtype=np.uint32)
    rep, freq, pres = (rng.random(rows).astype(np.float32) * s + o for s, o in ((0.5, 1.0), (0.5, 0.0), (0.5, 0.0)))
    if rows > 2:
        mask[2] = 0
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int64)).int().cuda()  # noqa: E731
    f32 = lambda a: torch.from_numpy(a.astype(np.float32)).cuda()  # noqa: E731
    best = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    out = ctx.logits_process(x.cuda(), best=best, history=i32(hist), history_len=i32(hlen), prompt_len=i32(plen), repetition=f32(rep),
                             frequency=f32(freq), presence=f32(pres), bias_ids=i32(ids), bias_values=f32(vals), bias_len=i32(blen),
                             mask=torch.from_numpy(mask.view(np.int32)).cuda())
    for r in range(rows):
        allowed = np.unpackbits(mask[r].view(np.uint8), bitorder="little")[:vocab].astype(bool)
        bias = [(int(i), float(v)) for i, v in zip(ids[r, :blen[r]], vals[r])]
        want = ref.logits(_np(x)[r], hist[r, :hlen[r]].tolist(), plen[r], float(rep[r]), float(freq[r]), float(pres[r]), bias, allowed)
        got = _np(out)[r]
        gone = ~np.isfinite(want)
        assert np.array_equal(got[gone], want[gone])
        # up to six FP32 roundings of values up to |x| * rep + 30 freq + pres + sum |bias|, then the output's
        size = np.abs(_np(x)[r]) * 1.5 + 30 * 0.5 + 0.5 + np.abs(vals[r]).sum()
        touched = np.isin(np.arange(vocab), np.concatenate([hist[r], ids[r]]))
        slack = np.where(touched, size * 10 * 2.0 ** -24, 0.0)
        assert np.all((np.abs(got - want)[~gone] <= (slack + _half_step(t) * (np.abs(want) + slack))[~gone]))
        top = np.flatnonzero(got == got.max()) if (got > -np.inf).any() else [-1]
        assert int(best[r]) == int(top[0])


def test_logits_in_place_strides_and_absent_parts(pkg, ctx):
    torch = _torch()
    wide = torch.randn(4, 1003, device="cuda").bfloat16()
    x = wide[:, 1:1000]
    keep = wide.clone()
    assert torch.equal(ctx.logits_process(x), x)
    best = torch.empty(4, dtype=torch.int32, device="cuda")
    mask = torch.zeros(4, 32, dtype=torch.int32, device="cuda")
    mask[:, 3] = 1 << 5
    out = ctx.logits_process(x, out=x, best=best, mask=mask)
    assert out.data_ptr() == x.data_ptr() and best.tolist() == [101] * 4
    assert torch.equal(wide[:, 0], keep[:, 0]) and torch.equal(wide[:, 1000:], keep[:, 1000:])
    assert torch.equal(x[:, 101], keep[:, 102]) and torch.isinf(x).sum() == 4 * 998
    # one row of logits for several masks, NaN and infinities, both zeros
    y = torch.tensor([[float("nan"), -float("inf"), 0.0, -0.0, -1.0, float("nan")]], device="cuda")
    m = torch.tensor([[63], [1], [56], [16]], dtype=torch.int32, device="cuda")
    best = torch.empty(4, dtype=torch.int32, device="cuda")
    got = ctx.logits_process(y.expand(4, -1), best=best, mask=m)
    assert best.tolist() == [2, -1, 3, 4] and torch.isnan(got[1, 0]) and not torch.isnan(got[2, 0])


def test_logits_feed_the_sampler(pkg, ctx):
    """Processed logits into the device sampler: only the allowed tokens come out."""
    torch = _torch()
    x = torch.zeros(1, 32256, device="cuda")
    x[0, 320:324] = torch.tensor([1.0, 0.5, 9.0, 0.25], device="cuda")  # the greatest of the four is not allowed
    mask = torch.zeros(1, 1008, dtype=torch.int32, device="cuda")
    mask[0, 10] = 0b1011
    best = torch.empty(1, dtype=torch.int32, device="cuda")
    out = ctx.logits_process(x[:, :32000], out=x[:, :32000], best=best, mask=mask)
    torch.cuda.synchronize()
    seen = {ctx.sample(out.data_ptr(), [], pkg.Sampler.make(1.0, 0.9, 1.0, seed * 0x9E3779B97F4A7C15 % 2 ** 64)) for seed in range(1, 40)}
    assert seen == {320, 321, 323} and best.item() == 320  # each has a probability above 0.22
    assert ctx.sample(out.data_ptr(), [], pkg.Sampler.make(0.0)) == best.item()
