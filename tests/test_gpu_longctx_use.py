"""The long-context serving operators as they are used: together, captured into
graphs, on several streams, with padded batches and with wrong arrays, and at
the ends of their ranges."""
import numpy as np
import pytest

import longctx_ref as ref
from test_gpu_longctx import Setup, _half_step, _np, _run_attention, _same_cache, _starts, _torch, _type

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(pkg):
    with pkg.Context(num_layers=1, kv_capacity=8) as c:
        yield c


# ------------------------------------------------------- wrong device arrays

@pytest.mark.parametrize("bad_id", [-1, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("name,q_lens,heads", [("bf16", [1, 1, 1], 4), ("f32", [5, 1, 3], 2), ("f16", [40, 1, 33], 4)])
def test_attention_skips_blocks_outside_the_pool(pkg, ctx, bad_id, name, q_lens, heads):
    lens = [300, 40, 77]
    s = Setup(pkg, lens, 2, 64, 16, "int8", 31)
    table = s.table.copy()
    table[0, 3] = table[0, 18] = bad_id
    table[2, 0] = bad_id
    _run_attention(pkg, ctx, s, q_lens, lens, heads, name, 0, table=table, bad="block id")
    table[0] = bad_id  # a sequence without a token left: zeros
    _, out = _run_attention(pkg, ctx, s, q_lens, lens, heads, name, 0, table=table, bad="block id")
    assert np.all(_np(out)[:q_lens[0]] == 0)


def test_long_sequences_skip_blocks_outside_the_pool(pkg, ctx):
    """Tokens shared by CTAs, and by clusters."""
    for lens in ([6000], [4097, 3, 5000, 900]):
        s = Setup(pkg, lens, 1, 128, 32, "e4m3", 37)
        table = s.table.copy()
        table[0, 7:90] = s.cache.blocks
        _run_attention(pkg, ctx, s, [1] * len(lens), lens, 2, "bf16", 0, table=table, bad="block id")


def test_append_read_and_evict_skip_blocks_outside_the_pool(pkg, ctx):
    torch = _torch()
    lens, q_lens = [100, 64, 37], [100, 20, 37]
    s = Setup(pkg, lens, 2, 64, 16, "int8", 41)
    table = s.table.copy()
    table[0, 2], table[2, 0] = -5, s.cache.blocks
    start = _starts(q_lens)
    k = torch.randn(157, 2, 64, device="cuda").bfloat16()
    want = s.ref()
    want.append((_np(k), _np(k)), start, lens, table)
    ctx.kv8_append(s.cache, k, k, s.dev(start), s.dev(lens), s.dev(table), 100)
    with pytest.raises(pkg.I4DError, match="block id"):
        ctx.ops_check()
    _same_cache(s.cache, want)
    out = torch.full((157, 2, 64), 7.0, device="cuda").bfloat16()
    ctx.kv8_read(s.cache, s.dev(start), s.dev(lens), s.dev(table), 100, 157, k_out=out)
    with pytest.raises(pkg.I4DError, match="block id"):
        ctx.ops_check()
    kept = np.ones(157, bool)
    kept[32:48] = kept[120:136] = False
    for b, n in enumerate(q_lens):
        for h in range(2):
            for i in range(n):
                if kept[start[b] + i]:
                    assert np.array_equal(_np(out)[start[b] + i, h], want.tokens(0, table[b], h, np.array([lens[b] - n + i]))[0])
    # eviction: the sequences beside it as without it, and nothing behind the pool
    w = torch.rand(3, 2, 100, device="cuda")
    before = (s.cache.k.clone(), s.cache.v.clone(), s.cache.k_scale.clone(), s.cache.v_scale.clone())
    good = pkg.KV8Cache(*(x.clone() for x in before))
    ctx.kv8_evict(good, s.dev(lens), s.dev(s.table), w.clone(), 30, 5, 100)
    ctx.ops_check()
    lo, _, _ = ctx.kv8_evict(s.cache, s.dev(lens), s.dev(table), w.clone(), 30, 5, 100)
    with pytest.raises(pkg.I4DError, match="block id"):
        ctx.ops_check()
    assert lo.tolist() == [30, 30, 30]
    for blk in s.table[1, :2]:
        assert torch.equal(s.cache.k[int(blk)], good.k[int(blk)]) and torch.equal(s.cache.v_scale[int(blk)], good.v_scale[int(blk)])
    untouched = [b for b in range(s.cache.blocks) if b not in set(table.ravel().tolist())]
    for b in untouched:
        assert torch.equal(s.cache.k[b], before[0][b]) and torch.equal(s.cache.v[b], before[1][b])


@pytest.mark.parametrize("q_start,lens", [([0, 3, 2, 4], [20, 30, 10]), ([0, 1, 2, 2 ** 31 - 1], [20, 30, 10]), ([-1, 1, 2, 4], [20, 30, 10]),
                                          ([0, 1, 2, 4], [20, 2 ** 31 - 1, 10]), ([0, 1, 2, 4], [20, -1, 10]), ([0, 1, 2, 4], [20, 49, 10]),
                                          ([0, 1, 2, 4], [20, 30, 1]), ([0, 1, 2, 9], [20, 30, 10])])
def test_sequences_out_of_range_are_skipped(pkg, ctx, q_start, lens):
    torch = _torch()
    s = Setup(pkg, [20, 30, 10], 2, 64, 16, "int8", 43)  # table rows of three blocks
    s.table = np.ascontiguousarray(s.table[:, :3])
    max_q, tokens, top = 2, 4, 48
    ok = [0 <= q_start[b] <= q_start[b + 1] <= tokens and q_start[b + 1] - q_start[b] <= min(max_q, lens[b]) and lens[b] <= top for b in range(3)]
    assert not all(ok)
    q = torch.randn(tokens, 4, 64, device="cuda").bfloat16()
    good_start, good_lens = list(q_start), list(lens)
    out = torch.full_like(q, 7.0)
    args = (s.dev(q_start), s.dev(lens), s.dev(s.table), max_q)
    weights = torch.zeros(3, 2, top, device="cuda")
    ctx.kv8_attention(s.cache, q, *args, top, out=out, weights=weights)
    with pytest.raises(pkg.I4DError, match="q_start or lengths"):
        ctx.ops_check()
    rows = torch.zeros(tokens, dtype=torch.bool)
    for b in range(3):
        if not ok[b]:
            assert torch.all(weights[b] == 0)
            continue
        a, e = good_start[b], good_start[b + 1]
        rows[a:e] = True
        alone = ctx.kv8_attention(s.cache, q[a:e], s.dev([0, e - a]), s.dev([good_lens[b]]), s.dev(s.table[b:b + 1]), max_q, top)
        assert torch.equal(out[a:e], alone)
    assert torch.all(out[~rows.cuda()] == 7)
    ctx.ops_check()
    before = s.cache.k.clone()
    k = torch.randn(tokens, 2, 64, device="cuda").bfloat16()
    ctx.kv8_append(s.cache, k, k, *args)
    with pytest.raises(pkg.I4DError, match="q_start or lengths"):
        ctx.ops_check()
    for b in range(3):
        if not ok[b]:
            for blk in s.table[b]:
                if blk not in s.table[[i for i in range(3) if ok[i]]]:
                    assert torch.equal(before[int(blk)], s.cache.k[int(blk)])
    back = torch.full((tokens, 2, 64), 7.0, device="cuda").bfloat16()
    ctx.kv8_read(s.cache, *args, tokens, k_out=back)
    with pytest.raises(pkg.I4DError, match="q_start or lengths"):
        ctx.ops_check()
    assert torch.all(back[~rows.cuda()] == 7)


def test_sync_reports_what_was_skipped_once(pkg):
    torch = _torch()
    with pkg.Context(num_layers=1, kv_capacity=8) as c:
        s = Setup(pkg, [20], 1, 64, 16, "int8", 44)
        k = torch.randn(1, 1, 64, device="cuda").bfloat16()
        c.kv8_append(s.cache, k, k, s.dev([0, 1]), s.dev([999]), s.dev(s.table), 1)
        torch.cuda.synchronize()
        with pytest.raises(pkg.I4DError, match="q_start or lengths"):
            c.sync()
        c.sync()


def test_another_thread_and_the_default_stream(pkg, ctx):
    import threading
    torch = _torch()
    s = Setup(pkg, [700], 2, 64, 16, "int8", 45)
    q = torch.randn(1, 8, 64, device="cuda").bfloat16()
    args = (s.dev([0, 1]), s.dev([700]), s.dev(s.table), 1, 700)
    want = ctx.kv8_attention(s.cache, q, *args)
    got = []

    def work():
        for _ in range(20):
            got.append(ctx.kv8_attention(s.cache, q, *args))

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(got) == 60 and all(torch.equal(x, want) for x in got)


def test_evict_skips_lengths_out_of_range(pkg, ctx):
    torch = _torch()
    s = Setup(pkg, [60, 60, 60], 1, 64, 16, "int8", 47)
    w = torch.rand(3, 1, 60, device="cuda")
    before, w0 = s.cache.k.clone(), w.clone()
    lo, keep, _ = ctx.kv8_evict(s.cache, s.dev([60, 61, -3]), s.dev(s.table), w, 20, 3, 60)
    with pytest.raises(pkg.I4DError, match="lengths"):
        ctx.ops_check()
    assert lo.tolist() == [20, 0, 0] and torch.all(keep[1:] == -1) and torch.equal(w[1:], w0[1:])
    for blk in s.table[1:, :4].ravel():
        assert torch.equal(before[int(blk)], s.cache.k[int(blk)])


# --------------------------------------------------- batches, streams, graphs

def test_padded_batch_and_empty_calls(pkg, ctx):
    """Sequences without rows or tokens at the end, rows behind the last one."""
    torch = _torch()
    s = Setup(pkg, [30, 17, 0, 0], 2, 64, 16, "int8", 53)
    _run_attention(pkg, ctx, s, [1, 4, 0, 0], [30, 17, 0, 0], 4, "bf16", 0, extra=9)
    _run_attention(pkg, ctx, s, [0, 1, 0, 0], [30, 17, 0, 0], 4, "f32", 0, extra=1, max_length=32)
    none = torch.empty(0, 4, 64, device="cuda").bfloat16()
    one = s.dev([0])
    assert ctx.kv8_attention(s.cache, none, one, s.dev([]), torch.empty(0, 3, dtype=torch.int32, device="cuda"), 1, 0).shape == (0, 4, 64)
    ctx.kv8_append(s.cache, none[:, :2], none[:, :2], one, s.dev([]), torch.empty(0, 3, dtype=torch.int32, device="cuda"), 0)
    table = pkg.RopeTable(64)
    assert ctx.rope(none, None, s.dev([]), table)[0].shape == (0, 4, 64)
    lo, keep, _ = ctx.kv8_evict(s.cache, s.dev([]), torch.empty(0, 3, dtype=torch.int32, device="cuda"), torch.empty(0, 2, 9, device="cuda"), 5, 1, 9)
    assert lo.shape == (0,) and keep.shape == (0, 2, 5)
    assert ctx.logits_process(torch.empty(0, 100, device="cuda")).shape == (0, 100)
    ctx.ops_check()


class Step:
    """One decode step of a batch: positions, the cache, attention with weights, logits.  All in buffers of its own."""

    def __init__(self, pkg, ctx, seed, lens, kv=2, group=4, dim=64, vocab=5000, rows=None):
        torch = _torch()
        self.ctx, n = ctx, rows or [1] * len(lens)
        self.s = Setup(pkg, [x + 40 for x in lens], kv, dim, 16, "int8", seed)
        g = torch.Generator().manual_seed(seed)
        self.start = _starts(n)
        total = int(self.start[-1])
        self.qkv = torch.randn(total, (group + 2) * kv, dim, generator=g).bfloat16().cuda()
        self.kv, self.heads = kv, kv * group
        self.pos, self.lens = torch.zeros(total, dtype=torch.int32).cuda(), self.s.dev(lens)
        self.q_start, self.table, self.max_q = self.s.dev(self.start), self.s.dev(self.s.table), max(n)
        self.top = max(lens) + 40
        self.rope = pkg.RopeTable(dim)
        self.out = torch.empty(total, self.heads, dim, dtype=torch.bfloat16, device="cuda")
        self.weights = torch.zeros(len(lens), kv, self.top, device="cuda")
        self.logits = torch.randn(total, vocab, generator=g).cuda()
        self.hist = torch.randint(0, vocab, (total, 50), generator=g, dtype=torch.int32).cuda()
        self.hlen = torch.full((total,), 50, dtype=torch.int32).cuda()
        self.rep = torch.full((total,), 1.25).cuda()
        self.best = torch.empty(total, dtype=torch.int32, device="cuda")
        self.processed = torch.empty_like(self.logits)

    def run(self):
        c, h = self.ctx, self.heads
        q, k, v = self.qkv[:, :h], self.qkv[:, h:h + self.kv], self.qkv[:, h + self.kv:]
        self.q, self.k = c.rope(q, k, self.pos, self.rope)
        c.kv8_append(self.s.cache, self.k, v, self.q_start, self.lens, self.table, self.max_q)
        c.kv8_attention(self.s.cache, self.q, self.q_start, self.lens, self.table, self.max_q, self.top, out=self.out, weights=self.weights)
        c.logits_process(self.logits, out=self.processed, best=self.best, history=self.hist, history_len=self.hlen, repetition=self.rep)

    def state(self):
        return [x.clone() for x in (self.out, self.weights, self.processed, self.best, self.s.cache.k, self.s.cache.v, self.s.cache.k_scale)]


def _shift(step, by):
    step.qkv.mul_(1 + by / 8)
    step.lens.add_(1)
    step.pos.add_(1 + by)


@pytest.mark.parametrize("lens", [[30, 1, 77], [2900], [5000, 9, 260, 1]])
def test_two_graphs_replay_like_eager_calls(pkg, ctx, lens):
    """Captured steps read their inputs at replay; two graphs alive at once, with eager calls between."""
    torch = _torch()
    eager, captured, other = (Step(pkg, ctx, 59, lens) for _ in range(3))
    for x in (eager, captured, other):
        x.run()
    graphs = []
    for x in (captured, other):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x.run()
        graphs.append(graph)
    for i in range(3):
        for x in (eager, captured, other):
            _shift(x, i)
        graphs[0].replay()
        eager.run()
        graphs[1].replay()
        for a, b, c in zip(eager.state(), captured.state(), other.state()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and torch.equal(a.view(torch.uint8), c.view(torch.uint8))
    ctx.ops_check()


def test_streams_side_by_side(pkg, ctx):
    torch = _torch()
    alone, a, b = (Step(pkg, ctx, 61, [4000, 20, 700]) for _ in range(3))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(4):
        for x, st in ((a, streams[0]), (b, streams[1])):
            with torch.cuda.stream(st):
                _shift(x, i)
                x.run()
    for i in range(4):
        _shift(alone, i)
        alone.run()
    torch.cuda.synchronize()
    for x, y, z in zip(alone.state(), a.state(), b.state()):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) and torch.equal(x.view(torch.uint8), z.view(torch.uint8))


@pytest.mark.parametrize("lens,rows", [([700, 3, 260], [1, 1, 1]), ([9000, 70], [1, 1]), ([300, 120], [90, 120])])
def test_results_are_repeatable(pkg, ctx, lens, rows):
    torch = _torch()
    first = None
    for _ in range(3):
        step = Step(pkg, ctx, 67, lens, rows=rows)
        step.run()
        state = step.state()
        first = first or state
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(first, state))


def test_own_workspace(pkg, ctx):
    """A workspace of the caller's, full of garbage, larger than needed, and one that is too small."""
    torch = _torch()
    s = Setup(pkg, [9000, 40], 1, 128, 32, "int8", 71)
    q = torch.randn(2, 2, 128, device="cuda").bfloat16()
    args = (s.dev([0, 1, 2]), s.dev([9000, 40]), s.dev(s.table), 1, 9000)
    want = ctx.kv8_attention(s.cache, q, *args)
    space = torch.full((1 << 26,), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(ctx.kv8_attention(s.cache, q, *args, workspace=space), want)
    with pytest.raises(pkg.I4DError, match="workspace"):
        ctx.kv8_attention(s.cache, q, *args, workspace=space[:64])
    with pytest.raises(pkg.I4DError, match="workspace"):
        ctx.kv8_attention(s.cache, q, *args, workspace=space[8:])
    w = torch.rand(2, 1, 9000, device="cuda")
    with pytest.raises(pkg.I4DError, match="workspace"):
        ctx.kv8_evict(s.cache, s.dev([9000, 40]), s.dev(s.table), w, 100, 10, 9000, workspace=space[:16])


def test_binding_refuses(pkg, ctx):
    torch = _torch()
    s = Setup(pkg, [20], 2, 64, 16, "int8", 73)
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()
    start, lens, table, rope = s.dev([0, 1]), s.dev([20]), s.dev(s.table), pkg.RopeTable(64)
    pos = s.dev([5])
    bad = [
        lambda: ctx.kv8_attention(s.cache, q.cpu(), start, lens, table, 1, 20),
        lambda: ctx.kv8_attention(s.cache, q.double(), start, lens, table, 1, 20),
        lambda: ctx.kv8_attention(s.cache, q[:, :3], start, lens, table, 1, 20),
        lambda: ctx.kv8_attention(s.cache, q[..., :48], start, lens, table, 1, 20),
        lambda: ctx.kv8_attention(s.cache, q[..., ::2], start, lens, table, 1, 20),
        lambda: ctx.kv8_attention(s.cache, q, start.long(), lens, table, 1, 20),
        lambda: ctx.kv8_attention(s.cache, q, start[:1], lens, table, 1, 20),
        lambda: ctx.kv8_attention(s.cache, q, start, lens, table[0], 1, 20),
        lambda: ctx.kv8_attention(s.cache, q, start, lens, table, 1, 2000),
        lambda: ctx.kv8_attention(s.cache, q, start, lens, table, 1, 20, out=q),
        lambda: ctx.kv8_attention(s.cache, q, start, lens, table, 1, 20, out=torch.empty_like(q).half()),
        lambda: ctx.kv8_attention(s.cache, q, start, lens, table, 1, 20, lse=torch.empty(1, 3, device="cuda")),
        lambda: ctx.kv8_attention(s.cache, q, start, lens, table, 1, 20, weights=torch.empty(1, 2, 19, device="cuda")),
        lambda: ctx.kv8_attention(s.cache, q, start, lens, table, 2 ** 40, 20),
        lambda: ctx.kv8_attention(s.cache, q.clone().requires_grad_(), start, lens, table, 1, 20),
        lambda: ctx.rope(q, None, s.dev([5, 6]), rope),
        lambda: ctx.rope(q, q[:, :2], pos, rope, q_out=q),
        lambda: ctx.rope(q.clone().requires_grad_(), None, pos, rope),
        lambda: ctx.kv8_append(s.cache, q[:, :1], q[:, :1], start, lens, table, 1),
        lambda: ctx.kv8_append(s.cache, q[:, :2], q[:, :2].half(), start, lens, table, 1),
        lambda: ctx.kv8_read(s.cache, start, lens, table, 1, -1),
        lambda: ctx.kv8_read(s.cache, start, lens, table, 1, 1, k_out=torch.empty(1, 2, 64, device="cuda")),
        lambda: ctx.kv8_evict(s.cache, lens, table, torch.zeros(1, 2, 20, device="cuda"), -1, 0, 20),
        lambda: ctx.kv8_evict(s.cache, lens, table, torch.zeros(1, 1, 20, device="cuda"), 5, 0, 20),
        lambda: ctx.kv8_evict(s.cache, lens, table, torch.zeros(1, 2, 20, device="cuda"), 5, 6, 20),
        lambda: ctx.logits_process(torch.zeros(2, 9, device="cuda"), history=torch.zeros(2, 3, dtype=torch.int32, device="cuda")),
        lambda: ctx.logits_process(torch.zeros(2, 9, device="cuda"), mask=torch.zeros(2, 0, dtype=torch.int32, device="cuda")),
        lambda: ctx.logits_process(torch.zeros(2, 9, device="cuda"), best=torch.zeros(3, dtype=torch.int32, device="cuda")),
        lambda: pkg.KV8Cache(s.cache.k, s.cache.v, s.cache.k_scale.half(), s.cache.v_scale),
        lambda: pkg.KV8Cache(s.cache.k.cpu(), s.cache.v.cpu(), s.cache.k_scale.cpu(), s.cache.v_scale.cpu()),
        lambda: pkg.KV8Cache.empty(4, 2, 16, 64, "int4"),
        lambda: pkg.RopeTable(65),
        lambda: pkg.RopeTable(64, scaling="other"),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(pkg.I4DError):
            f()
            pytest.fail(f"call {i} was accepted")
    with torch.no_grad():
        leaf = q.clone().requires_grad_()
        assert torch.equal(ctx.kv8_attention(s.cache, leaf, start, lens, table, 1, 20), ctx.kv8_attention(s.cache, q, start, lens, table, 1, 20))
    ctx.ops_check()


def test_closed_context(pkg):
    torch = _torch()
    c = pkg.Context(num_layers=1, kv_capacity=8)
    c.close()
    with pytest.raises(pkg.I4DError):
        c.logits_process(torch.zeros(1, 9, device="cuda"))


# ------------------------------------------------------- ends of the ranges

@pytest.mark.parametrize("name,kind", [("bf16", "int8"), ("f16", "e4m3")])
@pytest.mark.parametrize("group,n,length", [(5, 13, 70), (16, 8, 3000), (1, 129, 129), (8, 33, 2100), (1, 257, 1500), (64, 2, 500)])
def test_prompts_with_ragged_row_tiles(pkg, ctx, name, kind, group, n, length):
    """65 rows (a second tile of one), few rows over a long cache (its tokens shared by many CTAs), tiles of one row."""
    s = Setup(pkg, [length], 1, 128, 64, kind, 79 + n)
    _run_attention(pkg, ctx, s, [n], [length], group, name, 0)
    _run_attention(pkg, ctx, s, [n], [length], group, name, 200, max_length=min(length + 64, s.table.shape[1] * 64))


@pytest.mark.parametrize("batch,length,group", [(1, 1, 1), (1, 129, 1), (1, 1025, 8), (40, 300, 4), (300, 20, 1), (1, 20000, 1), (3, 9000, 16)])
def test_single_tokens_of_many_and_few_sequences(pkg, ctx, batch, length, group):
    rng = np.random.default_rng(batch + length)
    lens = [length] + rng.integers(1, length + 1, batch - 1).tolist()
    s = Setup(pkg, lens, 1, 64, 16, "int8", 83)  # up to 1250 blocks of a sequence
    _run_attention(pkg, ctx, s, [1] * batch, lens, group, "bf16", 0)


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("max_q,max_length", [(1, 300), (40, 400), (900, 4000), (5000, 20000)])
def test_bounds_far_above_what_the_sequences_have(pkg, ctx, name, max_q, max_length):
    """max_q and max_length only bound: with any of them the results are within the same bounds, whichever kernel they choose."""
    from test_gpu_longctx import _attention_bounds
    torch = _torch()
    lens, t = [300, 17, 64], _type(name)
    s = Setup(pkg, lens, 2, 128, 16, "int8", 113)
    table = np.zeros((3, max(s.table.shape[1], -(-max_length // 16))), np.int32)
    table[:, :s.table.shape[1]] = s.table
    start = _starts([1, 1, 1])
    g = torch.Generator().manual_seed(3)
    q, k = torch.randn(3, 4, 128, generator=g).to(t).cuda(), torch.randn(3, 2, 128, generator=g).to(t).cuda()
    want = s.ref()
    want.append((_np(k), _np(k)), start, lens, table)
    args = (s.dev(start), s.dev(lens), s.dev(table), max_q)
    ctx.kv8_append(s.cache, k, k, *args)
    _same_cache(s.cache, want)
    weights = torch.zeros(3, 2, max_length, device="cuda")
    lse = torch.empty(3, 4, device="cuda")
    out = ctx.kv8_attention(s.cache, q, *args, max_length, weights=weights, lse=lse)
    w_out, w_lse, sums, mag, size = ref.attention(want, _np(q), start, lens, table, 128 ** -0.5)
    b_out, b_lse, b_p = _attention_bounds(t, 128, w_out, mag, size, w_lse, 300)
    assert np.all(np.abs(_np(out) - w_out) <= b_out) and np.all(np.abs(_np(lse) - w_lse) <= b_lse)
    for b, n in enumerate(lens):  # two rows a head: their probabilities and two sums
        assert np.all(np.abs(_np(weights)[b, :, :n] - sums[b]) <= sums[b] * (b_p.max() + 2.0 ** -21))
        assert torch.all(weights[b, :, n:] == 0)
    back = ctx.kv8_read(s.cache, *args, 3)
    for b, n in enumerate(lens):
        for h in range(2):
            assert np.array_equal(_np(back[1])[b, h], want.tokens(1, table[b], h, np.array([n - 1]))[0])
    lo, keep, _ = ctx.kv8_evict(s.cache, args[1], args[2], weights, 50, 10, max_length)
    assert lo.tolist() == [50, 17, 50]
    ctx.ops_check()


@pytest.mark.parametrize("batch", [3000, 70000])
def test_thousands_of_sequences(pkg, ctx, batch):
    """Many sequences that share one block (read only), some without rows."""
    torch = _torch()
    s = Setup(pkg, [16], 1, 64, 16, "int8", 127)
    n = torch.ones(batch, dtype=torch.int32)
    n[::3] = 0
    start = torch.cat([torch.zeros(1, dtype=torch.int32), n.cumsum(0).int()]).cuda()
    total = int(start[-1])
    q = torch.randn(1, 2, 64, device="cuda").half()
    table = torch.full((1, 1), int(s.table[0, 0]), dtype=torch.int32, device="cuda").expand(batch, 1)
    lens = torch.full((batch,), 13, dtype=torch.int32, device="cuda")
    one = ctx.kv8_attention(s.cache, q, s.dev([0, 1]), s.dev([13]), s.dev(s.table), 1, 16)
    out = ctx.kv8_attention(s.cache, q.expand(total, -1, -1), start, lens, table, 1, 16)
    assert torch.equal(out, one.expand(total, -1, -1))
    ctx.ops_check()


@pytest.mark.parametrize("window", [1, 2, 15, 16, 64, 10 ** 9])
def test_windows(pkg, ctx, window):
    s = Setup(pkg, [3000, 64, 1], 1, 64, 32, "int8", 89)
    _run_attention(pkg, ctx, s, [1, 1, 1], [3000, 64, 1], 2, "bf16", window)
    _run_attention(pkg, ctx, s, [70, 64, 1], [3000, 64, 1], 2, "f16", window)


def test_scales_of_zero_and_below(pkg, ctx):
    """scale 0 weighs every token alike; a negative one turns the order around."""
    s = Setup(pkg, [200, 33], 1, 64, 16, "int8", 97)
    for scale in (0.0, -0.125):
        _run_attention(pkg, ctx, s, [1, 1], [200, 33], 2, "bf16", 0, scale=scale)
        _run_attention(pkg, ctx, s, [80, 33], [200, 33], 2, "bf16", 0, scale=scale)


@pytest.mark.parametrize("length,budget,recent", [(70001, 30000, 17), (66000, 65990, 0), (40000, 1, 1)])
def test_evict_long_rows(pkg, ctx, length, budget, recent):
    """Rows longer than the registers hold; in place and beside it the same."""
    torch = _torch()
    s = Setup(pkg, [length, 50], 1, 16, 128, "int8", 101)
    w = torch.from_numpy(s.rng.integers(0, 1000, (2, 1, length)).astype(np.float32)).cuda()
    w[1, :, 50:] = 0
    want = s.ref()
    lens_w, keep_w, w_w = want.evict(s.table, [length, 50], _np(w), budget, recent)
    other = pkg.KV8Cache(s.cache.k.clone(), s.cache.v.clone(), s.cache.k_scale.clone(), s.cache.v_scale.clone())
    beside = torch.full_like(w, 3.0)
    lo, keep, _ = ctx.kv8_evict(other, s.dev([length, 50]), s.dev(s.table), w, budget, recent, length, weights_out=beside)
    lo2, keep2, _ = ctx.kv8_evict(s.cache, s.dev([length, 50]), s.dev(s.table), w, budget, recent, length)
    ctx.ops_check()
    assert lo.tolist() == lo2.tolist() == lens_w and torch.equal(keep, keep2)
    assert np.array_equal(_np(keep[0, 0])[:lens_w[0]], keep_w[0][0]) and np.array_equal(_np(w), w_w)
    assert torch.equal(beside[0], w[0]) and torch.equal(beside[1, :, :50], w[1, :, :50])
    n = lens_w[0]
    for cache in (s.cache, other):
        got, sc = _np(cache.k), _np(cache.k_scale)
        for j in range(-(-n // 128)):
            part, blk = min(128, n - j * 128), s.table[0, j]
            assert np.array_equal(got[blk, :, :part], want.codes[0][blk, :, :part]) and np.array_equal(sc[blk], want.scale[0][blk])


def test_cache_beyond_32_bit_offsets(pkg, ctx):
    """Blocks 4.4 GB into the codes give what the same blocks of a small cache give."""
    torch = _torch()
    dim, bs, heads, far = 128, 128, 2, 136000  # 32 KB a block
    lens, q_lens = [300, 90], [3, 90]
    near = Setup(pkg, lens, heads, dim, bs, "int8", 109)
    low = -(-near.cache.blocks // 8) * 8
    big = pkg.KV8Cache.empty(far + low, heads, bs, dim, "int8")
    for a, b in ((big.k, near.cache.k), (big.v, near.cache.v), (big.k_scale, near.cache.k_scale), (big.v_scale, near.cache.v_scale)):
        a[far:far + near.cache.blocks] = b
    start, n = near.dev(_starts(q_lens)), near.dev(lens)
    tables = near.dev(near.table), near.dev(near.table + far)
    g = torch.Generator().manual_seed(5)
    rows = (torch.randn(93, 8, dim, generator=g)).bfloat16().cuda()
    results = []
    for cache, table in zip((near.cache, big), tables):
        ctx.kv8_append(cache, rows[:, :2], rows[:, 2:4], start, n, table, 90)
        weights = torch.zeros(2, heads, 300, device="cuda")
        out = [ctx.kv8_attention(cache, rows[:, :h], start, n, table, 90, 300, weights=weights) for h in (2, 8)]
        one = ctx.kv8_attention(cache, rows[:2], near.dev([0, 1, 2]), n, table, 1, 300, weights=weights)
        back = ctx.kv8_read(cache, start, n, table, 90, 93)
        lo, keep, _ = ctx.kv8_evict(cache, n, table, weights, 70, 10, 300)
        after = ctx.kv8_read(cache, near.dev([0, 70, 140]), lo, table, 70, 140)
        results.append([*out, one, *back, lo, keep, weights, *after])
    ctx.ops_check()
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert torch.all(big.k[:far].view(torch.int64) == 0)  # nothing below them was written


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_logits_with_more_ids_than_a_part_holds(pkg, ctx, name):
    torch = _torch()
    t, rows, vocab, n = _type(name), 2, 200003, 30000
    rng = np.random.default_rng(103)
    x = torch.from_numpy(rng.standard_normal((rows, vocab)) * 3).to(t)
    hist = rng.integers(0, vocab, (rows, n))
    hist[:, :5000] %= 100  # some tokens very often
    ids, vals = rng.permutation(vocab)[:700][None].repeat(rows, 0), rng.standard_normal((rows, 700)).astype(np.float32)
    ids[1, 600:] = ids[1, 5]  # in several rounds
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
    rep, freq, pres = (torch.tensor(v, dtype=torch.float32, device="cuda") for v in ([1.3, 1.0], [0.25, 0.0], [0.5, 0.125]))
    out = ctx.logits_process(x.cuda(), history=i32(hist), history_len=i32([n, n - 1]), prompt_len=i32([100, 0]), repetition=rep, frequency=freq,
                             presence=pres, bias_ids=i32(ids), bias_values=torch.from_numpy(vals).cuda(), bias_len=i32([700, 699]))
    for r, (m, p) in enumerate(((n, 100), (n - 1, 0))):
        count = [700, 699][r]
        y = _np(x)[r].copy()
        seen = np.unique(hist[r, :m])
        often = np.bincount(hist[r, p:m], minlength=vocab)
        f = [float(v[r]) for v in (rep, freq, pres)]
        y[seen] = np.where(y[seen] > 0, y[seen] / f[0], y[seen] * f[0])
        y -= often * f[1] + (often > 0) * f[2]
        np.add.at(y, ids[r, :count], vals[r, :count].astype(np.float64))
        # roundings: the quotient, frequency * n, two differences, up to 100 of the bias' sum and its addition
        size = np.abs(_np(x)[r]) * 1.3 + often * f[1] + 0.5 + np.bincount(ids[r, :count], np.abs(vals[r, :count]), vocab)
        slack = np.where(np.isin(np.arange(vocab), np.concatenate([seen, ids[r]])), size * 105 * 2.0 ** -24, 0.0)
        assert np.all(np.abs(_np(out)[r] - y) <= slack + _half_step(t) * (np.abs(y) + slack))


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_a_conversation(pkg, ctx, kind):
    """A prompt, decode steps, an eviction and more decode steps: rotary
    positions, cache, attention and eviction follow the 64-bit definitions from
    the same stored codes, and positions run on where the cache is cut."""
    torch = _torch()
    kv, group, dim, bs = 2, 4, 64, 16
    heads = kv * group
    lens = np.array([90, 33])
    s = Setup(pkg, [400, 400], kv, dim, bs, kind, 107)
    host = s.ref()
    rope, freq = pkg.RopeTable(dim, scaling="linear", factor=4.0), ref.frequencies(dim, scaling="linear", factor=4.0)
    weights, top = torch.zeros(2, kv, 200, device="cuda"), 200
    sums = np.zeros((2, kv, 200))
    steps = [list(lens)] + [[1, 1]] * 3
    seen = np.zeros(2, int)
    lengths = np.zeros(2, int)
    for turn, n in enumerate(steps + ["evict"] + [[1, 1]] * 3 + [[5, 70]]):
        if n == "evict":
            budget, recent = 48, 8
            order = _np(weights).copy()  # the weights that the device chooses by
            lo, keep, _ = ctx.kv8_evict(s.cache, s.dev(lengths), s.dev(s.table), weights, budget, recent, top)
            lens_w, keep_w, w_w = host.evict(s.table, lengths.tolist(), order, budget, recent)
            assert lo.tolist() == lens_w and np.array_equal(_np(weights), w_w)
            for b in range(2):
                for h in range(kv):
                    assert keep[b, h].tolist()[:lens_w[b]] == list(keep_w[b][h])
            sums = w_w.copy()
            lengths = np.array(lens_w)
            continue
        start = _starts(n)
        total = int(start[-1])
        qkv = torch.from_numpy(s.rng.standard_normal((total, heads + 2 * kv, dim)) * 1.5).bfloat16().cuda()
        pos = np.concatenate([seen[b] + np.arange(n[b]) for b in range(2)])
        seen += n
        lengths = lengths + n
        raw = _np(qkv)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        ctx.rope(q, k, s.dev(pos), rope, q_out=q, k_out=k)  # in place in the fused buffer
        turned = _np(qkv)
        exact = ref.rope(raw[:, :heads + kv], pos, freq, 1.0, True)
        # half a step of the output, and the FP32 rotation's error (2^-20 of the pair) before it
        pair = np.abs(raw[:, :heads + kv]) + np.abs(raw[:, :heads + kv].reshape(total, heads + kv, -1, 2)[..., ::-1].reshape(total, heads + kv, dim))
        assert np.all(np.abs(turned[:, :heads + kv] - exact) <= _half_step(torch.bfloat16) * np.abs(exact) + pair * 2.0 ** -20)
        assert np.array_equal(turned[:, heads + kv:], raw[:, heads + kv:])
        args = (s.dev(start), s.dev(lengths), s.dev(s.table), max(n))
        ctx.kv8_append(s.cache, k, v, *args)
        host.append((turned[:, heads:heads + kv], turned[:, heads + kv:]), start, lengths.tolist(), s.table)
        _same_tokens(s, host, lengths)
        out = ctx.kv8_attention(s.cache, q, *args, top, weights=weights)
        w_out, w_lse, w_sums, mag, size = ref.attention(host, turned[:, :heads], start, lengths.tolist(), s.table, dim ** -0.5)
        from test_gpu_longctx import _attention_bounds
        b_out, _, b_p = _attention_bounds(torch.bfloat16, dim, w_out, mag, size, w_lse, int(lengths.max()))
        assert np.all(np.abs(_np(out) - w_out) <= b_out)
        for b in range(2):
            m = lengths[b]
            sums[b, :, :m] += w_sums[b]
            # each step: probabilities off by the bound, a sum of n * group FP32 roundings
            assert np.all(np.abs(_np(weights)[b, :, :m] - sums[b, :, :m]) <= sums[b, :, :m] * (b_p.max() * 4 + (n[b] * group + turn + 1) * 2.0 ** -22) + 1e-7)
            assert torch.all(weights[b, :, m:] == 0)
        sums = np.where(np.arange(200) < lengths[:, None, None], _np(weights), 0.0)  # the next step adds to what the device has
    ctx.ops_check()


def _same_tokens(s, host, lengths):
    """The cache's tokens (what lies behind a sequence's end is free)."""
    for which, (codes, scale) in enumerate(((s.cache.k, s.cache.k_scale), (s.cache.v, s.cache.v_scale))):
        got, sc = _np(codes), _np(scale)
        for b, n in enumerate(lengths):
            for j in range(-(-n // s.bs)):
                part, blk = min(s.bs, n - j * s.bs), s.table[b, j]
                assert np.array_equal(sc[blk], host.scale[which][blk]) and np.array_equal(got[blk, :, :part], host.codes[which][blk, :, :part])
