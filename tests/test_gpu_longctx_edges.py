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
    `floor` of a row's greatest weight (a probability times a value scale) for each token that it sees."""
    torch = _torch()
    lse = torch.empty(n, q.shape[1], device="cuda")
    out = ctx.kv8_attention(s.cache, q, s.dev([0, n]), s.dev([length]), s.dev(s.table), n, length, scale=scale, lse=lse)
    ctx.ops_check()
    w_out, w_lse, _, mag, size = ref.attention(s.ref(), _np(q), [0, n], [length], s.table, scale)
    dx = size * ((s.dim / 16 + 6) * 2.0 ** -23 + 2.0 ** -22) + 2.0 ** -21
    p = 2 * dx + (2.0 ** -21 if q.dtype == torch.float32 else one_part) + length / 16 * 2.0 ** -23
    err = mag * p[..., None]
    if floor:
        c, blocks = s.ref(), s.table[0, np.arange(length) // s.bs]
        for row, a in np.ndindex(n, q.shape[1]):
            h, see = a // (q.shape[1] // s.heads), length - n + row + 1
            x = c.tokens(0, s.table[0], h, np.arange(see)) @ _np(q)[row, a] * scale
            greatest = (np.exp(x - w_lse[row, a]) * c.scale[1][blocks[:see], h]).max()
            err[row, a] += floor * greatest * np.abs(c.codes[1][blocks[:see], h, np.arange(see) % s.bs]).sum(0)
    # (FP16 values under 2^-14 lie 2^-24 apart)
    assert np.all(np.abs(_np(out) - w_out) <= err + _half(q.dtype) * (np.abs(w_out) + err) + (2.0 ** -25 if q.dtype == torch.float16 else 1e-30))
    assert np.all(np.abs(_np(lse) - w_lse) <= dx + length / 16 * 2.0 ** -23 + 2.0 ** -22 * (np.abs(w_lse) + 1))
    return out


def _half(t):
    return _torch().finfo(t).eps / 2


def _sinks(pkg, kind, length, at, seed):
    """Equal scores, but for the tokens of value 0 at `at` and every 100 behind it, so that all CTAs and warps have some;
    positive values, so that errors of equal probabilities add up."""
    torch = _torch()
    s = Setup(pkg, [length], 1, 64, 64, kind, seed)
    top = 12 if kind == "int8" else 10
    v = torch.from_numpy(s.rng.integers(6, top, s.cache.v.shape) * (8.0 if kind == "int8" else 16.0)).cuda()
    s.cache.k.zero_()
    s.cache.v.copy_(v.to(s.cache.v.dtype))
    for x in (s.cache.k_scale, s.cache.v_scale):
        x.fill_(1.0)
    where = np.arange(at, length, 100)
    block, slot = torch.from_numpy(s.table[0, where // 64].astype(np.int64)).cuda(), torch.from_numpy(where % 64).cuda()
    s.cache.k.view(torch.int8)[block, 0, slot, 0] = 64 if kind == "int8" else 0x68  # 64 as a code of either kind
    s.cache.v.view(torch.int8)[block, 0, slot] = 0
    return s


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kind,at", [("int8", 0), ("e4m3", 0), ("int8", 17), ("e4m3", 99)])
@pytest.mark.parametrize("down", [22.3, 26.7, 60.2])
def test_small_probabilities_of_a_long_tail(pkg, ctx, name, kind, at, down):
    """32441 tokens of 2^-down of the greatest weights, whose own values are 0: their relative precision is the output's.  Ones
    under FP16's range for 16-bit outputs too, though those of FP16 are then 0."""
    torch = _torch()
    s = _sinks(pkg, kind, 32769, at, 83)
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


@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("down", [15.0, 25.9, 31.0])
@pytest.mark.parametrize("at", [5, 40, 70, 100])
def test_probabilities_before_a_far_greater_one_in_prompts(pkg, ctx, name, kind, down, at):
    """One score of 2^down times the others', of value 0, anywhere among the first 128 tokens, and 32 of 2^(down / 4.8) before
    it, which do not raise their row's bound: the weights before it are scaled down with the sums, by less than FP16 holds."""
    torch = _torch()
    s = Setup(pkg, [128], 1, 64, 64, kind, 97)
    s.cache.k.zero_()
    s.cache.v.fill_(64)
    for x in (s.cache.k_scale, s.cache.v_scale):
        x.fill_(1.0)
    block, slot = int(s.table[0, at // 64]), at % 64
    s.cache.k[block, 0, slot - slot % 64:slot - slot % 64 + 32, 0] = 20  # the 32 tokens of a half's first part
    s.cache.k[block, 0, slot, 0] = 96
    s.cache.v.view(torch.int8)[block, 0, slot] = 0
    q = torch.zeros(1, 80, 64, device="cuda", dtype=_type(name))
    q[:, :, 0] = 1
    _attend(pkg, ctx, s, q, 1, 128, down * np.log(2) / 96, floor=2.0 ** -24)


# Above 64 rows a weight in FP16 is off by half a step of 2^-24 when it is made
# and once more, for each of its parts, when its row's bound is raised: 3 times
# 2^-25 at most, where the greatest is at least 2^8 (2^9, and the bound goes up to
# a whole power of two).
PROMPT_FLOOR = 1.5 * 2.0 ** -32


@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("kind,at", [("int8", 0), ("e4m3", 0), ("int8", 17), ("e4m3", 99)])
def test_small_probabilities_of_a_long_tail_in_prompts(pkg, ctx, name, kind, at):
    """As above for many rows, whose weights are right to 2^-32 of the greatest: 2^-9.7 of each here, 2^-2.7 if they lay at 1."""
    torch = _torch()
    s = _sinks(pkg, kind, 32769, at, 89)
    q = torch.zeros(1, 80, 64, device="cuda", dtype=_type(name))
    q[:, :, 0] = 1
    _attend(pkg, ctx, s, q, 1, 32769, 22.3 * np.log(2) / 64, floor=PROMPT_FLOOR)


@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_far_scores_of_many_draws_in_prompts(pkg, ctx, name, kind):
    torch = _torch()
    for seed in range(8):
        s = Setup(pkg, [300], 2, 128, 32, kind, 200 + seed)
        q = torch.randn(2, 80, 128, generator=torch.Generator().manual_seed(seed)).to(_type(name)).cuda()
        _attend(pkg, ctx, s, q, 2, 300, 0.2 * (1 + seed % 5), floor=PROMPT_FLOOR)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("name,heads", [("f16", 1), ("f16", 16), ("f16", 80), ("f16", 300), ("f32", 1), ("f32", 80)])
def test_probabilities_go_in_two_parts(pkg, ctx, name, kind, heads):
    """Two scores, 64 tokens each, whose values cancel to a thousandth: FP16 and FP32 outputs have their probabilities to 2^-21,
    however many rows a call has (in one part those of the lower score are off by 2^-11.7, all alike)."""
    torch = _torch()
    s = Setup(pkg, [128], 1, 64, 64, kind, 101)
    s.cache.k.zero_()
    for x in (s.cache.k_scale, s.cache.v_scale):
        x.fill_(1.0)
    for j in range(2):
        s.cache.k[int(s.table[0, j]), 0, :, 0] = 10 - j
        s.cache.v[int(s.table[0, j])] = ((100, -123) if kind == "int8" else (104, -128))[j]
    q = torch.zeros(1, heads, 64, device="cuda", dtype=_type(name))
    q[:, :, 0] = 1
    out = _attend(pkg, ctx, s, q, 1, 128, 0.3 * np.log(2), floor=PROMPT_FLOOR, one_part=2.0 ** -21)
    assert torch.all(out.abs() < 0.1)


# ------------------------------------------------------------------ errors

def test_no_report_is_lost_between_streams(pkg, ctx):
    """A wrong block id found on one stream while a check on another one takes what was found before: a check reports it."""
    torch = _torch()
    s = Setup(pkg, [20], 1, 64, 16, "int8", 103)
    k = torch.randn(1, 1, 64, device="cuda").bfloat16()
    start, long, fits, table = s.dev([0, 1]), s.dev([999]), s.dev([20]), s.dev(s.table)
    bad = torch.full_like(table, -1)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx.ops_check()
    for i in range(600):
        ctx.kv8_append(s.cache, k, k, start, long, table, 1)
        torch.cuda.current_stream().synchronize()
        with torch.cuda.stream(other):
            torch.cuda._sleep(200 * i)  # up to 60 us: before, in and behind the check
            ctx.kv8_append(s.cache, k, k, start, fits, bad, 1)
        with pytest.raises(pkg.I4DError, match="lengths") as first:
            ctx.ops_check()
        other.synchronize()
        if "block id" not in str(first.value):
            with pytest.raises(pkg.I4DError, match="block id"):
                ctx.ops_check()
    ctx.ops_check()


def test_sync_asks_for_reports_only_where_operators_ran(pkg):
    """A context of the decoder alone does not wait for the operators' error word; one whose operators are in a graph does."""
    import time
    torch = _torch()

    def micros(c):
        best = 1e9
        for _ in range(20):
            t = time.perf_counter()
            for _ in range(50):
                c.sync()
            best = min(best, (time.perf_counter() - t) / 50 * 1e6)
        return best

    with pkg.Context(num_layers=1, kv_capacity=8) as c:
        alone = micros(c)
        s = Setup(pkg, [20], 1, 64, 16, "int8", 107)
        k = torch.randn(1, 1, 64, device="cuda").bfloat16()
        lens = s.dev([20])
        args = (s.cache, k, k, s.dev([0, 1]), lens, s.dev(s.table), 1)
        c.kv8_append(*args)
        c.sync()
        assert alone < 0.8 * micros(c)  # one wait and one copy of three of each
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.kv8_append(*args)
        lens.fill_(999)
        graph.replay()
        torch.cuda.synchronize()
        with pytest.raises(pkg.I4DError, match="lengths"):
            c.sync()


def test_a_check_lets_other_threads_run(pkg, ctx):
    """What the stream of a check waits for may need Python: the check waits without holding it."""
    import threading
    import time
    torch = _torch()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    began = threading.Event()

    def check():
        with torch.cuda.stream(side):
            torch.cuda._sleep(10 ** 9)  # about half a second
            began.set()
            ctx.ops_check()

    t = threading.Thread(target=check)
    t.start()
    began.wait()
    ran = 0
    for _ in range(10):
        time.sleep(0.01)
        ran += t.is_alive()
    t.join()
    assert ran == 10
    ctx.ops_check()


# ------------------------------------------------------------- first calls

FIRST_CALLS = """
import importlib, os, sys, time
sys.path[:0] = [{root!r}, os.path.join({root!r}, "tests")]
import torch
from test_gpu_longctx import Setup
pkg = importlib.import_module("4pe_u250_b200")
torch.zeros(1, device="cuda")
with pkg.Context(num_layers=1, kv_capacity=8) as ctx:
    s = Setup(pkg, [300, 90], 2, 64, 16, "int8", 5)
    rope, mask = pkg.RopeTable(64), torch.randint(-2 ** 31, 2 ** 31 - 1, (2, 1000), dtype=torch.int32, device="cuda")
    start, lens, table = s.dev([0, 40, 80]), s.dev([300, 90]), s.dev(s.table)
    qkv = torch.randn(80, 8, 64, device="cuda").bfloat16()
    pos, weights = torch.arange(80, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, 300, device="cuda")
    logits, history = torch.randn(2, 32000, device="cuda"), torch.randint(0, 32000, (2, 9000), dtype=torch.int32, device="cuda")
    hlen, rep = s.dev([9000, 8000]), torch.full((2,), 1.2, device="cuda")
    state = (s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale, weights)
    before = [x.clone() for x in state]

    def run():
        q, k = ctx.rope(qkv[:, :4], qkv[:, 4:6], pos, rope)
        ctx.kv8_append(s.cache, k, qkv[:, 6:], start, lens, table, 40)
        few = ctx.kv8_attention(s.cache, q[:2], s.dev_start, lens, table, 1, 300)
        many = ctx.kv8_attention(s.cache, q, start, lens, table, 40, 300, weights=weights)
        n, keep, w = ctx.kv8_evict(s.cache, lens, table, weights, 64, 8, 300)
        back = ctx.kv8_read(s.cache, start, n, table, 40, 80)
        return [q, k, few, many, n, keep, *back, w, ctx.logits_process(logits, history=history, history_len=hlen, repetition=rep, mask=mask)]

    s.dev_start = s.dev([0, 1, 2])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # nothing of it has run in this process
        got = run()
    graph.replay()
    got = [x.clone() for x in got]
    for x, y in zip(state, before):
        x.copy_(y)
    want = run()
    ctx.ops_check()
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(got, want))
print("same")
"""


def test_first_calls_of_a_process_are_captured():
    """Kernels that have not been loaded yet, in a graph."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(root=root)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip().endswith("same"), out.stdout + out.stderr


def test_a_context_loads_no_operator(pkg):
    """Creating contexts for the decoder alone stays as quick as it was: the operators' kernels load when they are called."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = f"""
import importlib, sys, time
sys.path.insert(0, {root!r})
import torch
torch.zeros(1, device="cuda")
pkg = importlib.import_module("4pe_u250_b200")
pkg.load_library()
times = []
for _ in range(2):
    t = time.perf_counter()
    with pkg.Context(num_layers=1, kv_capacity=8):
        times.append(time.perf_counter() - t)
print(*times)
"""
    best = []
    for _ in range(3):
        out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
        assert out.returncode == 0, out.stderr
        first, second = map(float, out.stdout.split())
        best.append(first / second)
    # the first context of a process also loads the decoder's few kernels (7.6 ms after 3.6); with the operators' forty it took 35
    assert min(best) < 5


# ------------------------------------------------------------------ bounds

@pytest.mark.parametrize("max_q", [2 ** 31 - 1, 2 ** 31 - 16, 2 ** 30 + 1])
@pytest.mark.parametrize("bs", [16, 128])
def test_append_with_a_bound_of_new_tokens_near_32_bits(pkg, ctx, max_q, bs):
    """The bound says nothing that the rows do not: the same cache as with the greatest count."""
    torch = _torch()
    new = torch.randn(45, 2, 64, generator=torch.Generator().manual_seed(9)).cuda().bfloat16()
    found = []
    for most in (40, max_q):
        s = Setup(pkg, [300, 5], 2, 64, bs, "int8", 109)
        ctx.kv8_append(s.cache, new, new, s.dev([0, 40, 45]), s.dev([300, 5]), s.dev(s.table), most)
        found.append([x.clone() for x in (s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale)])
    ctx.ops_check()
    assert all(torch.equal(x, y) for x, y in zip(*found))
