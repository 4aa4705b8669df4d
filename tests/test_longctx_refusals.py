"""What the long-context operators refuse, on the CPU: the host side of the C
ABI with a context whose device does not exist, and the rules by which the
device skips wrong values of the arrays that it alone sees."""
import ctypes
import importlib
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, ERR_ARG, ERR_CUDA, ERR_SIZE = 0, 1, 3, 2
P, I, L, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float


def _struct(name, **fields):
    kinds = {}
    for kind, names in fields.items():
        kinds[kind] = names
    return type(name, (ctypes.Structure,), {"_fields_": _fields(kinds)})


def _fields(kinds):
    out = []
    for kind, names in kinds.items():
        c = {"p": P, "i": I, "l": L, "f": F, "z": ctypes.c_size_t}[kind[0]]
        out += [(n, c) for n in names.split()]
    return out


Rope = _struct("Rope", p="q k q_out k_out positions turns",
               l="q_stride q_head_stride k_stride k_head_stride q_out_stride q_out_head_stride k_out_stride k_out_head_stride",
               i="tokens q_heads k_heads dim rot_dim interleaved inverse dtype", f="magnitude", p2="stream")
Cache = _struct("Cache", p="k v k_scale v_scale", i="blocks heads block_tokens dim code")


class Append(ctypes.Structure):
    _fields_ = [("cache", Cache)] + _fields({"p": "k v", "l": "k_stride k_head_stride v_stride v_head_stride",
                                             "p2": "q_start lengths block_table", "l2": "table_stride",
                                             "i": "table_blocks batch tokens max_q dtype", "p3": "stream"})


class Read(ctypes.Structure):
    _fields_ = [("cache", Cache)] + _fields({"p": "k_out v_out q_start lengths block_table", "l": "table_stride",
                                             "i": "table_blocks batch tokens max_q", "p2": "stream"})


class Attention(ctypes.Structure):
    _fields_ = [("cache", Cache)] + _fields({
        "p": "q out lse weights", "l": "q_stride q_head_stride out_stride out_head_stride weights_stride",
        "p2": "q_start lengths block_table", "l2": "table_stride",
        "i": "table_blocks batch tokens heads max_q max_length window dtype", "f": "scale", "p3": "workspace",
        "z": "workspace_bytes", "p4": "stream"})


class Evict(ctypes.Structure):
    _fields_ = [("cache", Cache)] + _fields({
        "p": "weights weights_out", "l": "weights_stride weights_out_stride", "p2": "lengths lengths_out keep block_table",
        "l2": "table_stride", "i": "table_blocks batch budget recent max_length", "p3": "workspace", "z": "workspace_bytes",
        "p4": "stream"})


Logits = _struct("Logits", p="logits out best history history_len prompt_len repetition frequency presence bias_ids bias_values bias_len mask",
                 l="stride out_stride history_stride bias_stride mask_stride", i="rows vocab history_max bias_max dtype", p2="stream")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    build = importlib.import_module("4pe_u250_b200.build")
    inc = ["-I", os.path.join(ROOT, "include"), "-I", build.CSRC]
    obj = os.path.join(ROOT, "_build", "i4d_ops.o")
    tmp = tmp_path_factory.mktemp("stub")
    src = os.path.join(build.CSRC, "i4d_ops.cu")
    newest = max(os.path.getmtime(os.path.join(build.CSRC, f)) for f in os.listdir(build.CSRC) if f.endswith((".cuh", ".h")) or f == "i4d_ops.cu")
    if not os.path.exists(obj) or os.path.getmtime(obj) < newest:
        obj = str(tmp / "i4d_ops.o")
        subprocess.run([build.NVCC, *build.ARCH, "-std=c++17", "-Xcompiler", "-fPIC", *inc, "-c", src, "-o", obj], check=True)
    out = str(tmp / "stub.so")
    subprocess.run([build.NVCC, *build.ARCH, "-std=c++17", "-shared", "-Xcompiler", "-fPIC", *inc, os.path.join(ROOT, "tests", "longctx_stub.cpp"), obj,
                    "-o", out], check=True)
    x = ctypes.CDLL(out)
    x.stub_message.restype = ctypes.c_char_p
    return x


def _cache(**change):
    c = dict(k=0x10000000, v=0x20000000, k_scale=0x30000000, v_scale=0x31000000, blocks=8, heads=2, block_tokens=16, dim=64, code=0)
    c.update(change)
    return Cache(**c)


BATCH = dict(q_start=0x40000000, lengths=0x40001000, block_table=0x40002000, table_stride=4, table_blocks=4, batch=2, tokens=6, max_q=5)


def _rope(**change):
    a = dict(q=0x50000000, k=0x51000000, q_out=0x52000000, k_out=0x53000000, positions=0x40000000, turns=0x41000000,
             q_stride=256, q_head_stride=64, k_stride=128, k_head_stride=64, q_out_stride=256, q_out_head_stride=64,
             k_out_stride=128, k_out_head_stride=64, tokens=5, q_heads=4, k_heads=2, dim=64, rot_dim=64, interleaved=1,
             inverse=0, dtype=1, magnitude=1.0)
    a.update(change)
    return Rope(**a)


def _append(cache=None, **change):
    a = dict(BATCH, cache=_cache(**(cache or {})), k=0x50000000, v=0x51000000, k_stride=128, k_head_stride=64, v_stride=128, v_head_stride=64, dtype=1)
    a.update(change)
    return Append(**a)


def _read(cache=None, **change):
    a = dict(BATCH, cache=_cache(**(cache or {})), k_out=0x50000000, v_out=0x51000000)
    a.update(change)
    return Read(**a)


def _attention(cache=None, **change):
    a = dict(BATCH, cache=_cache(**(cache or {})), q=0x50000000, out=0x51000000, lse=0x52000000, weights=0x53000000, q_stride=256,
             q_head_stride=64, out_stride=256, out_head_stride=64, weights_stride=64, heads=4, max_length=64, window=0, dtype=1,
             scale=0.125, workspace=0x60000000, workspace_bytes=1 << 24)
    a.update(change)
    return Attention(**a)


def _evict(cache=None, **change):
    a = dict(cache=_cache(**(cache or {})), weights=0x50000000, weights_out=0x50000000, weights_stride=64, weights_out_stride=64,
             lengths=0x40000000, lengths_out=0x40001000, keep=0x40002000, block_table=0x40003000, table_stride=4, table_blocks=4,
             batch=2, budget=32, recent=8, max_length=64, workspace=0x60000000, workspace_bytes=1 << 20)
    a.update(change)
    return Evict(**a)


def _logits(**change):
    a = dict(logits=0x50000000, out=0x51000000, best=0x40000000, history=0x41000000, history_len=0x42000000, prompt_len=0x42001000,
             repetition=0x42002000, frequency=0x42003000, presence=0x42004000, bias_ids=0x43000000, bias_values=0x43100000,
             bias_len=0x42005000, mask=0x44000000, stride=1000, out_stride=1000, history_stride=50, bias_stride=9, mask_stride=32,
             rows=3, vocab=1000, history_max=50, bias_max=9, dtype=1)
    a.update(change)
    return Logits(**a)


def _call(lib, name, args):
    return getattr(lib, name)(P(0x1000), ctypes.byref(args))


MAKE = {"i4d_rope": _rope, "i4d_kv8_append": _append, "i4d_kv8_read": _read, "i4d_kv8_attention": _attention,
        "i4d_kv8_evict": _evict, "i4d_logits_process": _logits}

ACCEPTED = [
    ("i4d_rope", {}),
    ("i4d_rope", dict(k=0, k_out=0)),
    ("i4d_rope", dict(q_out=0x50000000, k_out=0x51000000)),  # in place
    # the q and k parts of one fused buffer [tokens][8][64], in place
    ("i4d_rope", dict(q_stride=512, k_stride=512, q_out_stride=512, k_out_stride=512, k=0x50000000 + 4 * 64 * 2,
                      q_out=0x50000000, k_out=0x50000000 + 4 * 64 * 2)),
    # q and k interleaved head by head [tokens][4][3][64], in place
    ("i4d_rope", dict(k_heads=4, q_stride=768, k_stride=768, q_out_stride=768, k_out_stride=768, q_head_stride=192, k_head_stride=192,
                      q_out_head_stride=192, k_out_head_stride=192, k=0x50000000 + 128, q_out=0x50000000, k_out=0x50000000 + 128)),
    ("i4d_rope", dict(q_stride=0)),  # one row for all tokens
    ("i4d_rope", dict(q_stride=64, q_head_stride=5 * 64, q_out_stride=64, q_out_head_stride=5 * 64)),  # [heads][tokens]
    ("i4d_rope", dict(tokens=1, q_heads=1, k=0, q_out_stride=0, q_out_head_stride=0)),
    ("i4d_kv8_append", {}),
    ("i4d_kv8_append", dict(k_stride=0, v=0x50000000)),
    ("i4d_kv8_read", {}),
    ("i4d_kv8_attention", {}),
    ("i4d_kv8_attention", dict(lse=0, weights=0, workspace=0, workspace_bytes=0, max_length=64)),
    ("i4d_kv8_attention", dict(cache=dict(v=0x10000000))),  # values that are the keys
    # out into the same rows' other half
    ("i4d_kv8_attention", dict(q_stride=512, out_stride=512, out=0x50000000 + 512)),
    ("i4d_kv8_evict", {}),
    ("i4d_kv8_evict", dict(weights_out=0x59000000, weights_out_stride=100)),
    ("i4d_logits_process", {}),
    ("i4d_logits_process", dict(out=0x50000000)),
    ("i4d_logits_process", dict(stride=0)),
    ("i4d_logits_process", dict(best=0, history=0, history_len=0, prompt_len=0, repetition=0, frequency=0, presence=0, bias_ids=0, bias_values=0,
                                bias_len=0, mask=0)),
]

NOTHING = [
    ("i4d_rope", dict(tokens=0)), ("i4d_kv8_append", dict(batch=0)), ("i4d_kv8_append", dict(tokens=0)), ("i4d_kv8_append", dict(max_q=0)),
    ("i4d_kv8_read", dict(tokens=0)), ("i4d_kv8_attention", dict(batch=0)), ("i4d_kv8_attention", dict(tokens=0)), ("i4d_kv8_evict", dict(batch=0)),
    ("i4d_logits_process", dict(rows=0)),
]

REFUSED = [
    ("i4d_rope", dict(dtype=3), "dtype"), ("i4d_rope", dict(dtype=-1), "dtype"), ("i4d_rope", dict(tokens=-1), "tokens"),
    ("i4d_rope", dict(q_heads=0), "q_heads"), ("i4d_rope", dict(dim=0), "dim"), ("i4d_rope", dict(dim=4097), "dim"),
    ("i4d_rope", dict(rot_dim=66), "rot_dim"), ("i4d_rope", dict(rot_dim=3), "rot_dim"), ("i4d_rope", dict(rot_dim=0), "rot_dim"),
    ("i4d_rope", dict(q=0), "null"), ("i4d_rope", dict(q_out=0), "null"), ("i4d_rope", dict(positions=0), "null"), ("i4d_rope", dict(turns=0), "null"),
    ("i4d_rope", dict(k_out=0), "k_out"), ("i4d_rope", dict(q=0x50000001), "misaligned"), ("i4d_rope", dict(turns=0x41000004), "misaligned"),
    ("i4d_rope", dict(q_stride=-1), "stride"), ("i4d_rope", dict(q_out_stride=255), "q_out"), ("i4d_rope", dict(k_out_head_stride=63), "k_out"),
    ("i4d_rope", dict(q_out=0x50000002), "q_out overlaps q"), ("i4d_rope", dict(q_out=0x50000000, q_out_stride=512), "q_out overlaps q"),
    ("i4d_rope", dict(q_out=0x51000000), "q_out overlaps k"), ("i4d_rope", dict(k_out=0x50000000), "k_out overlaps q"),
    ("i4d_rope", dict(k_out=0x52000000), "q_out overlaps k_out"), ("i4d_rope", dict(k_out=0x52000100), "q_out overlaps k_out"),
    ("i4d_rope", dict(positions=0x52000010), "positions"), ("i4d_rope", dict(turns=0x53000000), "turns"),
    # a fused buffer whose k starts one head early
    ("i4d_rope", dict(q_stride=512, k_stride=512, q_out_stride=512, k_out_stride=512, k=0x50000000 + 3 * 64 * 2, q_out=0x50000000,
                      k_out=0x50000000 + 3 * 64 * 2), "overlaps"),
    ("i4d_rope", dict(dim=65, rot_dim=64, q_stride=260, k_stride=260, q_out_stride=260, k_out_stride=260, q_head_stride=65, k_head_stride=65,
                      q_out_head_stride=65, k_out_head_stride=65), "even"),
    ("i4d_kv8_append", dict(cache=dict(k=0)), "null"), ("i4d_kv8_append", dict(cache=dict(blocks=0)), "blocks"),
    ("i4d_kv8_append", dict(cache=dict(block_tokens=8)), "block_tokens"), ("i4d_kv8_append", dict(cache=dict(block_tokens=256)), "block_tokens"),
    ("i4d_kv8_append", dict(cache=dict(dim=24)), "dim"), ("i4d_kv8_append", dict(cache=dict(dim=272)), "dim"),
    ("i4d_kv8_append", dict(cache=dict(code=2)), "code"), ("i4d_kv8_append", dict(cache=dict(k=0x10000008)), "alignment"),
    ("i4d_kv8_append", dict(cache=dict(v_scale=0x31000002)), "alignment"), ("i4d_kv8_append", dict(cache=dict(v=0x10000010)), "overlaps"),
    ("i4d_kv8_append", dict(cache=dict(v_scale=0x30000000)), "overlaps"), ("i4d_kv8_append", dict(k=0x10000000), "overlaps k"),
    ("i4d_kv8_append", dict(lengths=0x30000000), "overlaps lengths"), ("i4d_kv8_append", dict(k=0), "null"), ("i4d_kv8_append", dict(v=0), "null"),
    ("i4d_kv8_append", dict(v=0x51000001), "misaligned"), ("i4d_kv8_append", dict(k_stride=-1), "stride"), ("i4d_kv8_append", dict(q_start=0), "null"),
    ("i4d_kv8_append", dict(batch=-1), "negative"), ("i4d_kv8_append", dict(max_q=-1), "negative"), ("i4d_kv8_append", dict(table_blocks=-1), "negative"),
    ("i4d_kv8_append", dict(lengths=0x40001002), "alignment"), ("i4d_kv8_append", dict(dtype=7), "dtype"),
    ("i4d_kv8_append", dict(batch=1 << 30, cache=dict(heads=64)), "too many"),
    ("i4d_kv8_read", dict(k_out=0), "alignment"), ("i4d_kv8_read", dict(v_out=0x51000008), "alignment"), ("i4d_kv8_read", dict(v_out=0x50000000), "overlaps"),
    ("i4d_kv8_read", dict(k_out=0x20000000), "overlaps"), ("i4d_kv8_read", dict(block_table=0), "null"),
    ("i4d_kv8_attention", dict(heads=3), "heads"), ("i4d_kv8_attention", dict(heads=0), "heads"), ("i4d_kv8_attention", dict(max_length=65), "max_length"),
    ("i4d_kv8_attention", dict(max_length=-1), "max_length"), ("i4d_kv8_attention", dict(window=-1), "window"),
    ("i4d_kv8_attention", dict(scale=float("nan")), "scale"), ("i4d_kv8_attention", dict(scale=float("inf")), "scale"),
    ("i4d_kv8_attention", dict(q=0), "null"), ("i4d_kv8_attention", dict(out=0), "null"), ("i4d_kv8_attention", dict(q=0x50000001), "misaligned"),
    ("i4d_kv8_attention", dict(lse=0x52000002), "misaligned"), ("i4d_kv8_attention", dict(out=0x50000000), "out overlaps q"),
    ("i4d_kv8_attention", dict(out=0x50000010), "out overlaps q"), ("i4d_kv8_attention", dict(out_stride=255), "rows of out"),
    ("i4d_kv8_attention", dict(q_stride=-256), "stride"), ("i4d_kv8_attention", dict(weights_stride=63), "weights"),
    ("i4d_kv8_attention", dict(lse=0x53000000), "overlaps"), ("i4d_kv8_attention", dict(workspace=0x51000000), "overlaps"),
    ("i4d_kv8_attention", dict(workspace=0x10000000), "overlaps"), ("i4d_kv8_attention", dict(weights=0x50000000), "overlaps q"),
    ("i4d_kv8_attention", dict(workspace=0), "workspace"), ("i4d_kv8_attention", dict(workspace=0x60000008), "workspace"),
    ("i4d_kv8_attention", dict(cache=dict(blocks=1 << 26, block_tokens=128)), "2^31"), ("i4d_kv8_attention", dict(dtype=9), "dtype"),
    ("i4d_kv8_evict", dict(budget=0), "budget"), ("i4d_kv8_evict", dict(recent=33), "recent"), ("i4d_kv8_evict", dict(recent=-1), "recent"),
    ("i4d_kv8_evict", dict(max_length=65, weights_stride=65, weights_out_stride=65), "max_length"), ("i4d_kv8_evict", dict(weights_stride=63), "weights"),
    ("i4d_kv8_evict", dict(weights_out_stride=63, weights_out=0x59000000), "weights"), ("i4d_kv8_evict", dict(weights_out_stride=80), "overlaps"),
    ("i4d_kv8_evict", dict(weights_out=0x50000004), "overlaps"), ("i4d_kv8_evict", dict(lengths_out=0x40000000), "overlaps"),
    ("i4d_kv8_evict", dict(keep=0x40000004), "overlaps"), ("i4d_kv8_evict", dict(keep=0x50000000), "overlaps"), ("i4d_kv8_evict", dict(keep=0), "null"),
    ("i4d_kv8_evict", dict(workspace=0), "workspace"), ("i4d_kv8_evict", dict(workspace=0x40003000), "overlaps"),
    ("i4d_kv8_evict", dict(cache=dict(v=0x10000000)), "overlaps"), ("i4d_kv8_evict", dict(weights=0x50000002), "alignment"),
    ("i4d_kv8_evict", dict(batch=-1), "batch"),
    ("i4d_logits_process", dict(vocab=0), "vocab"), ("i4d_logits_process", dict(rows=-1), "rows"), ("i4d_logits_process", dict(dtype=4), "dtype"),
    ("i4d_logits_process", dict(logits=0), "null"), ("i4d_logits_process", dict(out=0x51000001), "misaligned"),
    ("i4d_logits_process", dict(out_stride=999), "out_stride"), ("i4d_logits_process", dict(stride=-1), "stride"),
    ("i4d_logits_process", dict(out=0x50000002), "overlaps"), ("i4d_logits_process", dict(out=0x50000000, out_stride=1008), "overlaps"),
    ("i4d_logits_process", dict(history_len=0), "history"), ("i4d_logits_process", dict(history=0), "history"),
    ("i4d_logits_process", dict(history_max=-1), "history"), ("i4d_logits_process", dict(bias_values=0), "bias"),
    ("i4d_logits_process", dict(bias_len=0), "bias"), ("i4d_logits_process", dict(bias_stride=-1), "bias"),
    ("i4d_logits_process", dict(mask_stride=-1), "mask"), ("i4d_logits_process", dict(best=0x50000004), "best overlaps"),
    ("i4d_logits_process", dict(best=0x51000004), "overlaps best"), ("i4d_logits_process", dict(mask=0x51000000), "overlaps mask"),
    ("i4d_logits_process", dict(history=0x41000002), "alignment"),
]


@pytest.mark.parametrize("name,change", ACCEPTED)
def test_accepted_calls_reach_the_device(lib, name, change):
    assert _call(lib, name, MAKE[name](**change)) == ERR_CUDA, lib.stub_message()


@pytest.mark.parametrize("name,change", NOTHING)
def test_empty_calls_do_nothing(lib, name, change):
    assert _call(lib, name, MAKE[name](**change)) == OK, lib.stub_message()


@pytest.mark.parametrize("name,change,says", REFUSED)
def test_refused(lib, name, change, says):
    assert _call(lib, name, MAKE[name](**change)) == ERR_ARG, lib.stub_message()
    assert says in lib.stub_message().decode(), lib.stub_message()


@pytest.mark.parametrize("name", MAKE)
def test_null_context_and_arguments(lib, name):
    f = getattr(lib, name)
    assert f(P(0), ctypes.byref(MAKE[name]())) == ERR_ARG
    assert f(P(0x1000), P(0)) == ERR_ARG


@pytest.mark.parametrize("name,make", [("i4d_kv8_attention", _attention), ("i4d_kv8_evict", _evict)])
def test_workspace_sizes(lib, name, make):
    need = ctypes.c_size_t()
    a = make()
    assert getattr(lib, name + "_workspace")(P(0x1000), ctypes.byref(a), ctypes.byref(need)) == OK
    assert need.value > 0
    a.workspace_bytes = need.value
    assert _call(lib, name, a) == ERR_CUDA
    a.workspace_bytes = need.value - 1
    assert _call(lib, name, a) == ERR_SIZE
    assert getattr(lib, name + "_workspace")(P(0x1000), ctypes.byref(a), P(0)) == ERR_ARG
    assert getattr(lib, name + "_workspace")(P(0), ctypes.byref(a), ctypes.byref(need)) == ERR_ARG


# The rules by which the device skips what it finds in the arrays; every access
# to rows, tables, cache and weights is made with values that passed them.

def test_sequences_that_pass_stay_in_bounds(lib):
    top = 2 ** 31 - 1
    values = (-top - 1, -1, 0, 1, 3, 4, 5, 16, 63, 64, 65, top)
    for q0 in values:
        for q1 in values:
            for n in values:
                for blocks in (0, 4, 1 << 30):
                    ok = lib.stub_seq_ok(q0, q1, n, 5, 4, blocks, 16)
                    want = 0 <= q0 <= q1 <= 5 and q1 - q0 <= 4 and q1 - q0 <= n <= min(16 * blocks, 1 << 30)
                    assert bool(ok) == want, (q0, q1, n, blocks)


def test_blocks_and_lengths_that_pass_stay_in_bounds(lib):
    top = 2 ** 31 - 1
    for x in (-top - 1, -1, 0, 1, 7, 8, 9, top):
        assert bool(lib.stub_block_ok(x, 8)) == (0 <= x < 8)
        assert bool(lib.stub_length_ok(x, 8)) == (0 <= x <= 8)


def test_binding_refuses_before_it_calls(pkg):
    """Tensors that are not on the context's GPU, wrong types and counts of arguments: the library is not reached."""
    torch = pytest.importorskip("torch")
    longctx = importlib.import_module("4pe_u250_b200.longctx")
    ops = longctx.ops()
    q, pos, turns = torch.zeros(2, 3, 8), torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(pkg.I4DError, match="q is not on GPU 0"):
        ops.rope(1, 0, q, None, pos, turns, 8, 1.0, True, False, None, None)
    with pytest.raises(pkg.I4DError, match="not a tensor"):
        ops.rope(1, 0, 7, None, pos, turns, 8, 1.0, True, False, None, None)
    with pytest.raises(pkg.I4DError, match="arguments"):
        ops.rope(1, 0, q)
    with pytest.raises(TypeError):
        ops.rope("x", 0, q, None, pos, turns, 8, 1.0, True, False, None, None)
    with pytest.raises(pkg.I4DError, match="KV8Cache"):
        ops.kv8_append(1, 0, None, q, q, pos, pos, pos, 1)
    with pytest.raises(pkg.I4DError, match="gradient"):
        ops.logits_process(1, 0, torch.zeros(1, 9, requires_grad=True), *[None] * 12)
    with pytest.raises(pkg.I4DError):
        pkg.KV8Cache(*(torch.zeros(2, 1, 16, 16, dtype=torch.int8) for _ in range(2)), *(torch.zeros(2, 1) for _ in range(2)))
    for bad in (dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=258), dict(rot_dim=8, base=1.0), dict(rot_dim=8, base=float("nan")),
                dict(rot_dim=8, scaling="linear", factor=0.5), dict(rot_dim=2, scaling="base", factor=2.0),
                dict(rot_dim=8, scaling="parts", factor=2.0, low=4.0, high=4.0), dict(rot_dim=8, scaling="cubic")):
        with pytest.raises(pkg.I4DError):
            pkg.rope_frequencies(**bad)
