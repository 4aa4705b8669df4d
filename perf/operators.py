"""Measured cases of the long-context serving operators: rotary positions, the
block-scaled 8-bit KV cache (append, read, attention, eviction) and the logits
processor.  `run` computes each in elementary torch operations (own = False) or
through the package's public calls (own = True); `exact` restates it in 64 bits.
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

_BF16, _F16, _F32 = "bf16", "f16", "f32"
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_TOP = {"int8": 127.0, "e4m3": 448.0}


def listed():
    return [
        # One decode step of a small batch: latency of the smallest call (this model's 32 heads of 128, adjacent pairs).
        {"name": "rope_decode", "op": "rope", "tokens": 5, "heads": 32, "kv_heads": 32, "dim": 128, "rot": 128,
         "pairs": "adjacent", "scaling": "none", "factor": 1.0, "top": 4096, "type": _BF16},
        # A long prompt's chunk at far positions: half-split pairs, half of each head rotated, frequencies scaled by parts.
        {"name": "rope_prompt", "op": "rope", "tokens": 8191, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 64,
         "pairs": "split", "scaling": "parts", "factor": 16.0, "top": 131072, "type": _BF16},
        # One new token for each of a ragged batch of streams.
        {"name": "append_decode", "op": "append", "batch": 48, "q_lo": 1, "q_hi": 1, "len_lo": 17, "len_hi": 2047,
         "kv_heads": 8, "dim": 128, "block": 32, "codes": "int8", "type": _BF16},
        # Prompt chunks of odd lengths that begin and end inside blocks.
        {"name": "append_prompt", "op": "append", "batch": 6, "q_lo": 501, "q_hi": 1531, "len_lo": 1601, "len_hi": 6007,
         "kv_heads": 8, "dim": 128, "block": 64, "codes": "e4m3", "type": _F32},
        # One stream at this repository's KV capacity of 2048, one query row per head.
        {"name": "decode_one", "op": "attention", "batch": 1, "q_lo": 1, "q_hi": 1, "len_lo": 2047, "len_hi": 2047,
         "heads": 32, "kv_heads": 32, "dim": 128, "block": 32, "codes": "int8", "type": _F32, "window": 0, "weights": False},
        # A serving batch of ragged contexts with shared heads: the cache's bytes are the time.
        {"name": "decode_batch", "op": "attention", "batch": 24, "q_lo": 1, "q_hi": 1, "len_lo": 301, "len_hi": 32749,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "codes": "int8", "type": _BF16, "window": 0, "weights": False},
        # Decode that also keeps the accumulated weights an eviction reads.
        {"name": "decode_weights", "op": "attention", "batch": 4, "q_lo": 1, "q_hi": 1, "len_lo": 9001, "len_hi": 24571,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 16, "codes": "e4m3", "type": _F16, "window": 0, "weights": True},
        # A prompt chunk over an earlier context: the matrix products are the time.
        {"name": "prompt_chunk", "op": "attention", "batch": 2, "q_lo": 1537, "q_hi": 2048, "len_lo": 6151, "len_hi": 8192,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "codes": "int8", "type": _BF16, "window": 0, "weights": False},
        # One stream's cache of 2048 slots brought back to half.
        {"name": "evict_one", "op": "evict", "batch": 1, "len_lo": 2047, "len_hi": 2047, "kv_heads": 32, "dim": 128,
         "block": 32, "codes": "int8", "budget": 1024, "recent": 256},
        # A batch of long contexts cut to one budget; the shortest is under it and stays.
        {"name": "evict_batch", "op": "evict", "batch": 4, "len_lo": 4001, "len_hi": 40009, "kv_heads": 8, "dim": 128,
         "block": 64, "codes": "e4m3", "budget": 8192, "recent": 1000},
        # The logits of one greedy step of this model: penalties over the history, a few biases, a grammar mask.
        {"name": "logits_one", "op": "logits", "rows": 1, "vocab": 32000, "history": 1500, "bias": 20, "mask": True,
         "type": _F32},
        # A batch over a large vocabulary.
        {"name": "logits_batch", "op": "logits", "rows": 192, "vocab": 128001, "history": 6000, "bias": 300, "mask": True,
         "type": _BF16},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], evenly spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "decode", "decode", "prompt", "evict", "logits"])
    block, codes = rng.choice([16, 32, 64, 128]), rng.choice(["int8", "e4m3"])
    dtype = rng.choice([_BF16, _F16, _F32])
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        heads = rng.choice([4, 8, 16, 32])
        tokens = _spread(rng, 1, 8191 * 40 * 128 // (dim * heads * 2) // (2 if dtype == _F32 else 1))
        scaling = rng.choice(["none", "linear", "base", "parts"])
        return {"op": op, "tokens": tokens, "heads": heads, "kv_heads": heads // rng.choice([1, 2, 4]), "dim": dim,
                "rot": rng.choice([dim, dim // 2, 16]), "pairs": rng.choice(["adjacent", "split"]), "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice([2.0, 8.0, 32.0]),
                "top": _spread(rng, 1000, 2000000), "type": dtype}
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 16, 32])
    if op == "append":
        most = 6007 * 8 * 128 * 3
        hi = _spread(rng, 1, max(1, min(1600, most // (kv_heads * dim * 4))))
        batch = _spread(rng, 1, max(1, min(64, most // (kv_heads * dim * (hi + block)))))
        before = _spread(rng, 1, 3000)
        return {"op": op, "batch": batch, "q_lo": (hi + 1) // 2, "q_hi": hi, "len_lo": hi + before // 2,
                "len_hi": hi + before, "kv_heads": kv_heads, "dim": dim, "block": block, "codes": codes, "type": dtype}
    if op == "decode":
        hi = _spread(rng, 1, 32749)
        batch = _spread(rng, 1, max(1, min(64, 24 * 32749 * 8 * 128 // 2 // (hi * kv_heads * dim))))
        return {"op": "attention", "batch": batch, "q_lo": 1, "q_hi": rng.choice([1, 1, 1, 3]), "len_lo": max(3, hi // 3),
                "len_hi": max(3, hi), "heads": kv_heads * rng.choice([1, 2, 4, 8] if kv_heads <= 8 else [1, 2]),
                "kv_heads": kv_heads, "dim": dim, "block": block, "codes": codes, "type": dtype,
                "window": rng.choice([0, 0, 500]), "weights": rng.random() < 0.4}
    if op == "prompt":
        group = rng.choice([1, 2, 4, 8])
        kv_heads = rng.choice([1, 2, 4, 8])
        hi = _spread(rng, 40, 1500)
        length = hi + _spread(rng, 1, 6000)
        most = 2 * 1792 * 7000 * 32 * 128
        batch = _spread(rng, 1, max(1, min(4, most // (hi * length * kv_heads * group * dim * (4 if dtype == _F32 else 2)))))
        return {"op": "attention", "batch": batch, "q_lo": (hi + 1) // 2, "q_hi": hi, "len_lo": (length + hi) // 2,
                "len_hi": length, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "block": block,
                "codes": codes, "type": dtype, "window": rng.choice([0, 0, 777]), "weights": rng.random() < 0.3}
    if op == "evict":
        hi = _spread(rng, 200, 40009)
        batch = _spread(rng, 1, max(1, min(16, 4 * 22000 * 8 * 128 // (hi * kv_heads * dim))))
        budget = max(16, int(hi * rng.uniform(0.1, 0.8)) if batch * kv_heads * dim * hi < 4 * 8192 * 8 * 128 else hi // 5)
        return {"op": op, "batch": batch, "len_lo": max(1, hi // 2), "len_hi": hi, "kv_heads": kv_heads, "dim": dim,
                "block": block, "codes": codes, "budget": budget, "recent": rng.choice([0, 1, budget // 4, budget])}
    vocab = rng.choice([32000, _spread(rng, 1000, 256000)])
    rows = _spread(rng, 1, max(1, min(256, 192 * 128001 // (2 if dtype == _F32 else 1) // vocab)))
    return {"op": "logits", "rows": rows, "vocab": vocab, "history": _spread(rng, 1, 6000), "bias": rng.choice([0, 5, 300]),
            "mask": rng.random() < 0.7, "type": dtype}


# ------------------------------------------------------------------ inputs

def _lengths(case, seed):
    """Query lengths and cache lengths of the sequences: spread evenly between the case's ends, in an order of the seed's."""
    n = case["batch"]
    step = lambda lo, hi: [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]  # noqa: E731
    both = list(zip(step(case.get("q_lo", 0), case.get("q_hi", 0)), step(case["len_lo"], case["len_hi"])))
    both = [(q, max(q, k)) for q, k in both]
    if seed is not None:
        random.Random(seed).shuffle(both)
    return [q for q, _ in both], [k for _, k in both]


def _starts(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).cuda()


def _cache(case, lens, g):
    """A pool of blocks in an order of the seed's, the tables, and codes whose values are about normal, with a scale of its own for each block and head."""
    bs, heads, dim = case["block"], case["kv_heads"], case["dim"]
    counts = [-(-k // bs) for k in lens]
    pool, wide = sum(counts) + 3, max(counts)
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), wide, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    made = {}
    low = -6 if case["codes"] == "int8" else -8
    for name in ("k", "v"):
        scale = torch.exp2(torch.randint(low, low + 3, (pool, heads), generator=g, device="cuda").float())
        codes = torch.empty(pool, heads, bs, dim, dtype=_CODES[case["codes"]], device="cuda")
        for part in torch.arange(pool, device="cuda").split(max(1, (1 << 26) // (heads * bs * dim))):
            x = torch.randn(len(part), heads, bs, dim, generator=g, device="cuda") / scale[part, :, None, None]
            x = x.clamp(-_TOP[case["codes"]], _TOP[case["codes"]])
            codes[part[0]:part[-1] + 1] = (x.round() if case["codes"] == "int8" else x).to(codes.dtype)
        made[name], made[name + "_scale"] = codes, scale
    return {**made, "table": table, "lengths": torch.tensor(lens, dtype=torch.int32, device="cuda")}


def _frequencies(case):
    """Radians a position, in 64 bits, and what the rotated values are multiplied by."""
    rot, base, f = case["rot"], 10000.0, case["factor"]
    i = np.arange(0, rot, 2, dtype=np.float64)
    if case["scaling"] == "base":
        base *= f ** (rot / (rot - 2.0))
    inv = base ** (-i / rot)
    if case["scaling"] == "linear":
        inv = inv / f
    if case["scaling"] == "parts":
        keep = np.clip((4096.0 * inv / (2.0 * math.pi) - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        inv = inv * (keep + (1.0 - keep) / f)
        return inv, 0.1 * math.log(f) + 1.0
    return inv, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    t = _TYPES.get(case.get("type"))
    if case["op"] == "rope":
        n = case["tokens"]
        s["q"] = torch.randn(n, case["heads"], case["dim"], generator=g, device="cuda").to(t)
        s["k"] = torch.randn(n, case["kv_heads"], case["dim"], generator=g, device="cuda").to(t)
        first = torch.randint(0, max(1, case["top"] - n), (1,), generator=g, device="cuda")
        s["positions"] = (first + torch.arange(n, device="cuda")).to(torch.int32)
        return s
    if case["op"] == "logits":
        n, v, h = case["rows"], case["vocab"], case["history"]
        s["logits"] = (torch.randn(n, v, generator=g, device="cuda") * 3.0).to(t)
        # Token ids of a text: small ones far more often, so that many repeat.
        s["history"] = (torch.rand(n, h, generator=g, device="cuda").pow(4) * v).to(torch.int32).clamp(0, v - 1)
        part = torch.rand(n, 2, generator=g, device="cuda")
        s["history_len"] = (part[:, 0] * 0.5 * h + 0.5 * h + 0.5).to(torch.int32).clamp(1, h)
        s["prompt_len"] = (part[:, 1] * s["history_len"]).to(torch.int32)
        s["repetition"] = 1.0 + 0.3 * torch.rand(n, generator=g, device="cuda")
        s["frequency"] = 0.5 * torch.rand(n, generator=g, device="cuda")
        s["presence"] = 0.5 * torch.rand(n, generator=g, device="cuda")
        if case["bias"]:
            ids = torch.rand(n, v, generator=g, device="cuda").topk(case["bias"], dim=1).indices
            s["bias_ids"] = ids.to(torch.int32)
            s["bias_values"] = 4.0 * torch.randn(n, case["bias"], generator=g, device="cuda")
            s["bias_len"] = torch.randint(0, case["bias"] + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        if case["mask"]:
            words = -(-v // 32)
            s["mask"] = torch.randint(-2 ** 31, 2 ** 31, (n, words), generator=g, device="cuda").to(torch.int32)
        s["out"] = torch.empty_like(s["logits"])
        s["best"] = torch.empty(n, dtype=torch.int32, device="cuda")
        return s
    q_lens, lens = _lengths(case, seed)
    s.update(_cache(case, lens, g))
    s["max_length"] = max(lens)
    n, wide = len(lens), s["table"].shape[1] * case["block"]
    if case["op"] == "evict":
        s["weights"] = torch.rand(n, case["kv_heads"], wide, generator=g, device="cuda").pow(8) * 3.0
        s["weights"] *= (torch.arange(wide, device="cuda") < s["lengths"][:, None])[:, None]
        kept = [min(k, case["budget"]) for k in lens]
        s["read_start"], s["read_most"], s["read_tokens"] = _starts(kept), max(kept), sum(kept)
        s["weights_out"] = torch.zeros_like(s["weights"])
        s["lengths_out"] = torch.zeros_like(s["lengths"])
        s["keep"] = torch.zeros(n, case["kv_heads"], case["budget"], dtype=torch.int32, device="cuda")
        return s
    s["q_start"], s["max_q"], total = _starts(q_lens), max(q_lens), sum(q_lens)
    if case["op"] == "append":
        spread = torch.exp(0.5 * torch.randn(total, case["kv_heads"], 1, generator=g, device="cuda"))
        for name in ("new_k", "new_v"):
            x = torch.randn(total, case["kv_heads"], case["dim"], generator=g, device="cuda")
            s[name] = (x * spread).to(t)
        # What is read back: the new tokens and those before them in the first block.
        read = [q + (k - q) % case["block"] for q, k in zip(q_lens, lens)]
        s["read_start"], s["read_most"], s["read_tokens"] = _starts(read), max(read), sum(read)
        return s
    s["q"] = (torch.randn(total, case["heads"], case["dim"], generator=g, device="cuda") * 1.5).to(t)
    s["out"], s["lse"] = torch.empty_like(s["q"]), torch.empty(total, case["heads"], device="cuda")
    if case["weights"]:
        s["weights"] = torch.rand(n, case["kv_heads"], wide, generator=g, device="cuda")
        s["weights"] *= (torch.arange(wide, device="cuda") < s["lengths"][:, None])[:, None]
    return s


# ------------------------------------------------------------- plain forms

def _rotate(x, c, s, pairs, rot):
    if pairs == "adjacent":
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        return torch.cat([torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2), x[..., rot:]], dim=-1)
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], dim=-1)


def _plain_rope(s):
    case = s["case"]
    inv, size = _frequencies(case)
    angle = s["positions"].double()[:, None] * torch.tensor(inv, device="cuda")
    c, d = ((f(angle) * size).float()[:, None, :] for f in (torch.cos, torch.sin))
    return [_rotate(x.float(), c, d, case["pairs"], case["rot"]).to(x.dtype) for x in (s["q"], s["k"])]


def _power_scale(top, most):
    """The least power of two s, not under 2^-126, with top <= most * s."""
    frac, exp = torch.frexp(top / most)
    return torch.exp2((torch.where(frac == 0.5, exp - 1, exp)).clamp(min=-126).float()).where(top > 0, torch.tensor(2.0 ** -126, device="cuda"))


def _coded(x, codes):
    """Whole codes of x / scale: rounded to the nearest, ties to even."""
    return (x.round() if codes == "int8" else x).clamp(-_TOP[codes], _TOP[codes]).to(_CODES[codes])


def _places(start, lengths, total):
    """Sequence and position of each of the last tokens that `start` counts out."""
    t = torch.arange(total, device="cuda")
    b = torch.searchsorted(start[1:].long(), t, right=True)
    return b, lengths.long()[b] - (start.long()[b + 1] - start.long()[b]) + t - start.long()[b]


def _plain_read(s, start, lengths, total):
    bs = s["case"]["block"]
    b, p = _places(start, lengths, total)
    blk = s["table"].long()[b, p // bs]
    return [(s[n][blk, :, p % bs].float() * s[n + "_scale"][blk][..., None]).bfloat16() for n in ("k", "v")]


def _plain_append(s):
    case = s["case"]
    bs, kind, total = case["block"], case["codes"], s["new_k"].shape[0]
    b, p = _places(s["q_start"], s["lengths"], total)
    blk = s["table"].long()[b, p // bs]
    before = s["lengths"].long() - (s["q_start"][1:] - s["q_start"][:-1]).long()
    first = s["table"].long().gather(1, (before // bs)[:, None])[:, 0]  # each sequence's first block that is written
    fill = before % bs
    for name in ("k", "v"):
        codes, scale, x = s[name], s[name + "_scale"], s["new_" + name].float()
        old = scale[first]
        top = torch.zeros_like(scale).scatter_reduce_(0, blk[:, None].expand(-1, scale.shape[1]), x.abs().amax(-1), "amax")
        new = _power_scale(top, _TOP[kind])
        had = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, first[fill > 0], True)
        new = torch.where(had[:, None], torch.maximum(new, scale), new)
        touched = torch.zeros_like(had).index_fill_(0, blk, True)
        scale.copy_(torch.where(touched[:, None], new, scale))
        held = codes[first]
        again = _coded(held.float() * (old / scale[first])[..., None, None], kind)
        keep = (torch.arange(bs, device="cuda") < fill[:, None])[:, None, :, None]
        bits = torch.where(keep, again.view(torch.int8), held.view(torch.int8))
        codes.view(torch.int8)[first] = bits
        codes.view(torch.int8)[blk, :, p % bs] = _coded(x / scale[blk][..., None], kind).view(torch.int8)
    k, v = _plain_read(s, s["read_start"], s["lengths"], s["read_tokens"])
    return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attention(s):
    case = s["case"]
    bs, heads, kv, dim = case["block"], case["heads"], case["kv_heads"], case["dim"]
    n, wide = s["table"].shape[0], s["table"].shape[1] * case["block"]
    total, most, group = s["q"].shape[0], s["max_q"], heads // kv
    b, p = _places(s["q_start"], s["lengths"], total)
    row = torch.arange(total, device="cuda") - s["q_start"].long()[b]
    q = torch.zeros(n, most, kv, group, dim, device="cuda")
    q[b, row] = s["q"].float().view(total, kv, group, dim)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, kv, group * most, dim)
    blk = s["table"].long()
    k, v = ((s[x][blk].float() * s[x + "_scale"][blk][..., None, None]).transpose(1, 2).reshape(n, kv, wide, dim) for x in ("k", "v"))
    score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    score = score.view(n, kv, group, most, wide)
    at = (s["lengths"].long() - (s["q_start"][1:] - s["q_start"][:-1]).long())[:, None] + torch.arange(most, device="cuda")
    j = torch.arange(wide, device="cuda")
    seen = (j <= at[..., None]) & (j < s["lengths"][:, None, None])
    seen &= (torch.arange(most, device="cuda") < (s["q_start"][1:] - s["q_start"][:-1])[:, None])[..., None]
    if case["window"]:
        seen &= j > at[..., None] - case["window"]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    prob = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    size = prob.sum(-1, keepdim=True)
    prob = prob / torch.where(size == 0, torch.ones_like(size), size)
    out = torch.matmul(prob.view(n, kv, group * most, wide), v).view(n, kv, group, most, dim)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, most, heads, dim)[b, row].to(s["q"].dtype)
    lse = (top + torch.log(size))[..., 0].permute(0, 3, 1, 2).reshape(n, most, heads)[b, row]
    if case["weights"]:
        s["weights"] += prob.sum((2, 3))
        return {"out": out, "lse": lse, "weights": s["weights"]}
    return {"out": out, "lse": lse}


def _plain_evict(s):
    case = s["case"]
    bs, kind, budget, recent = case["block"], case["codes"], case["budget"], case["recent"]
    w, n = s["weights"], s["table"].shape[0]
    wide = w.shape[2]
    j = torch.arange(wide, device="cuda")
    lens = s["lengths"].long()[:, None, None]
    always = (j >= lens - recent) | (lens <= budget)
    order = torch.where(always, math.inf, w).masked_fill(j >= lens, -math.inf)
    order = torch.sort(order, dim=2, descending=True, stable=True).indices[:, :, :min(budget, wide)]
    kept = lens.clamp(max=budget)
    i = torch.arange(order.shape[2], device="cuda")
    order = torch.where(i < kept, order, wide).sort(2).values
    valid = order < wide
    src = order.clamp(max=wide - 1)
    rows = torch.arange(n, device="cuda")[:, None, None]
    h = torch.arange(case["kv_heads"], device="cuda")[None, :, None]
    blk = s["table"].long()[rows, src // bs]
    i = torch.arange(-(-order.shape[2] // bs) * bs, device="cuda")
    to = s["table"].long()[:, :i.numel() // bs]
    for name in ("k", "v"):
        codes, scale = s[name], s[name + "_scale"]
        held = codes.view(torch.int8)[blk, h, src % bs].view(codes.dtype)
        from_scale = torch.where(valid, scale[blk, h], 0.0)
        padded = torch.nn.functional.pad(from_scale, (0, i.numel() - order.shape[2])).unflatten(2, (-1, bs))
        new = padded.amax(3)  # [n, heads, blocks]
        each = new.repeat_interleave(bs, 2)[:, :, :order.shape[2]]
        moved = _coded(held.float() * torch.where(valid, from_scale / each, 0.0)[..., None], kind).view(torch.int8)
        ri, hi, ii = valid.nonzero(as_tuple=True)
        codes.view(torch.int8)[to[ri, ii // bs], hi, ii % bs] = moved[ri, hi, ii]
        rj, hj, jj = (new > 0).nonzero(as_tuple=True)
        scale[to[rj, jj], hj] = new[rj, hj, jj]
    s["lengths_out"].copy_(kept[:, 0, 0])
    s["keep"].fill_(-1)
    s["keep"][:, :, :order.shape[2]] = torch.where(valid, order, -1).int()
    s["weights_out"].zero_()
    s["weights_out"][:, :, :order.shape[2]] = torch.where(valid, w.gather(2, src), 0.0)
    k, v = _plain_read(s, s["read_start"], s["lengths_out"], s["read_tokens"])
    return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"], "keep": s["keep"],
            "lengths": s["lengths_out"], "weights": s["weights_out"]}


def _plain_logits(s):
    case = s["case"]
    x = s["logits"].float()
    j = torch.arange(case["history"], device="cuda")
    ids = s["history"].long()
    seen, made = (torch.zeros_like(x, dtype=torch.int32) for _ in range(2))
    valid = j < s["history_len"][:, None]
    seen.scatter_add_(1, ids, valid.int())
    made.scatter_add_(1, ids, (valid & (j >= s["prompt_len"][:, None])).int())
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * made.float()
    x = x - torch.where(made > 0, s["presence"][:, None], 0.0)
    if case["bias"]:
        live = torch.arange(case["bias"], device="cuda") < s["bias_len"][:, None]
        x = x + torch.zeros_like(x).scatter_add_(1, s["bias_ids"].long(), torch.where(live, s["bias_values"], 0.0))
    if case["mask"]:
        v = torch.arange(case["vocab"], device="cuda")
        x = torch.where((s["mask"][:, v // 32] >> (v % 32)) & 1 != 0, x, -math.inf)
    s["out"].copy_(x)
    y = s["out"].float()
    top = y.amax(1, keepdim=True)
    v = torch.arange(case["vocab"], device="cuda")
    s["best"].copy_(torch.where(y == top, v, case["vocab"]).amin(1).where(top[:, 0] > -math.inf, -1))
    return {"logits": s["out"], "best": s["best"]}


_PLAIN = {"rope": _plain_rope, "append": _plain_append, "attention": _plain_attention, "evict": _plain_evict, "logits": _plain_logits}

# ------------------------------------------------------- the package's calls

_held = {}


def _package():
    """The package and one context on this GPU, as a program keeps them."""
    if not _held:
        _held["pkg"] = importlib.import_module("4pe_u250_b200")
        _held["ctx"] = _held["pkg"].Context(device=torch.cuda.current_device(), num_layers=1, kv_capacity=8)
    return _held["pkg"], _held["ctx"]


def _own_rope(s):
    pkg, ctx = _package()
    case = s["case"]
    if "rotary" not in s:
        s["rotary"] = pkg.RopeTable(case["rot"], base=10000.0, scaling=case["scaling"], factor=case["factor"],
                                    original_length=4096, low=1.0, high=32.0,
                                    magnitude=0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "parts" else 1.0)
    return ctx.rope(s["q"], s["k"], s["positions"], s["rotary"], interleaved=case["pairs"] == "adjacent")


def _own_cache(s):
    pkg, ctx = _package()
    if "cache" not in s:
        s["cache"] = pkg.KV8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return ctx, s["cache"]


def _own_append(s):
    ctx, cache = _own_cache(s)
    ctx.kv8_append(cache, s["new_k"], s["new_v"], s["q_start"], s["lengths"], s["table"], s["max_q"])
    k, v = ctx.kv8_read(cache, s["read_start"], s["lengths"], s["table"], s["read_most"], s["read_tokens"])
    return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _own_attention(s):
    ctx, cache = _own_cache(s)
    ctx.kv8_attention(cache, s["q"], s["q_start"], s["lengths"], s["table"], s["max_q"], s["max_length"],
                      window=s["case"]["window"], out=s["out"], lse=s["lse"], weights=s.get("weights"))
    return {x: s[x] for x in ("out", "lse", "weights") if x in s}


def _own_evict(s):
    ctx, cache = _own_cache(s)
    ctx.kv8_evict(cache, s["lengths"], s["table"], s["weights"], s["case"]["budget"], s["case"]["recent"], s["max_length"],
                  lengths_out=s["lengths_out"], keep=s["keep"], weights_out=s["weights_out"])
    k, v = ctx.kv8_read(cache, s["read_start"], s["lengths_out"], s["table"], s["read_most"], s["read_tokens"])
    return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"], "keep": s["keep"],
            "lengths": s["lengths_out"], "weights": s["weights_out"]}


def _own_logits(s):
    _, ctx = _package()
    ctx.logits_process(s["logits"], out=s["out"], best=s["best"], history=s["history"], history_len=s["history_len"],
                       prompt_len=s["prompt_len"], repetition=s["repetition"], frequency=s["frequency"],
                       presence=s["presence"], bias_ids=s.get("bias_ids"), bias_values=s.get("bias_values"),
                       bias_len=s.get("bias_len"), mask=s.get("mask"))
    return {"logits": s["out"], "best": s["best"]}


_OWN = {"rope": _own_rope, "append": _own_append, "attention": _own_attention, "evict": _own_evict, "logits": _own_logits}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------------- work

def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}.get(case.get("type"))
    if case["op"] == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["dim"] * size + 4 * case["tokens"], "flops": 3 * n * case["rot"]}
    if case["op"] == "logits":
        n = case["rows"] * case["vocab"]
        ids = case["rows"] * (case["history"] * 0.75 * 4 + case["bias"] * 0.5 * 8)
        return {"bytes": 2 * n * size + ids + (n / 8 if case["mask"] else 0), "flops": 4 * n}
    q_lens, lens = _lengths(case, None)
    row = case["kv_heads"] * case["dim"]
    scales = lambda tokens: 2 * 4 * case["kv_heads"] * sum(-(-t // case["block"]) for t in tokens)  # noqa: E731
    if case["op"] == "append":  # new values in, codes out, then the touched blocks' tokens read back
        read = [q + (k - q) % case["block"] for q, k in zip(q_lens, lens)]
        n = sum(q_lens)
        return {"bytes": 2 * row * (n * (size + 1) + (sum(read) - n) * 2 + sum(read) * 3) + 3 * scales(read), "flops": 4 * row * n}
    if case["op"] == "evict":  # kept codes in and out, the weights, then the kept tokens read back
        kept = [min(k, case["budget"]) for k in lens]
        cut = [m for m, k in zip(kept, lens) if m < k]
        return {"bytes": 2 * row * (2 * sum(cut) + 3 * sum(kept)) + 4 * case["kv_heads"] * (sum(lens) + 2 * sum(kept)) + 3 * scales(kept),
                "flops": 2 * row * sum(cut)}
    pairs, tokens = 0, 0
    for q, k in zip(q_lens, lens):
        w = case["window"] or k
        pairs += sum(min(k - q + i + 1, w) for i in range(q))
        tokens += min(k, w + q - 1)
    out = 2 * sum(q_lens) * case["heads"] * case["dim"] * size + 4 * sum(q_lens) * case["heads"]
    return {"bytes": 2 * row * tokens + scales(lens) + out + (8 * case["kv_heads"] * tokens if case["weights"] else 0),
            "flops": 4 * case["dim"] * case["heads"] * pairs}


# ------------------------------------------- the definitions, in 64 bits

def _exact_rope(s):
    case = s["case"]
    rot, half = case["rot"], case["rot"] // 2
    inv, size = _frequencies(case)
    z = torch.polar(torch.full((len(s["positions"]), half), size, dtype=torch.float64, device="cuda"),
                    torch.outer(s["positions"].double(), torch.tensor(inv, device="cuda")))
    found = []
    for x in (s["q"].double(), s["k"].double()):
        y = x.clone()
        if case["pairs"] == "adjacent":
            y[..., :rot] = torch.view_as_real(torch.view_as_complex(x[..., :rot].reshape(*x.shape[:2], half, 2).contiguous()) * z[:, None]).flatten(-2)
        else:
            w = torch.complex(x[..., :half].contiguous(), x[..., half:rot].contiguous()) * z[:, None]
            y[..., :half], y[..., half:rot] = w.real, w.imag
        found.append(y)
    return found


def _round_code(y, kind):
    """The nearest code's value for y in 64 bits, ties to even: whole numbers, or three fraction bits down to steps of 2^-9."""
    y = y.clamp(-_TOP[kind], _TOP[kind])
    if kind == "int8":
        return torch.round(y)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_append(s):
    case = s["case"]
    bs, kind = case["block"], case["codes"]
    starts, lens, table, reads = (s[x].tolist() for x in ("q_start", "lengths", "table", "read_start"))
    found = {}
    for name in ("k", "v"):
        value = s[name].double() * s[name + "_scale"].double()[..., None, None]
        scale = s[name + "_scale"].double()
        back = []
        for i, length in enumerate(lens):
            new = s["new_" + name][starts[i]:starts[i + 1]].double()
            first = length - new.shape[0]
            for j in range(first // bs, -(-length // bs)):
                lo, hi, blk = max(first, j * bs), min(length, (j + 1) * bs), table[i][j]
                part = new[lo - first:hi - first].transpose(0, 1)  # [heads, tokens, dim]
                top = part.abs().amax((1, 2)).cpu().numpy() / _TOP[kind]
                want = np.exp2(np.maximum(np.ceil(np.log2(np.maximum(top, 2.0 ** -140))), -126.0))
                at = torch.tensor(want, device="cuda")
                if lo > j * bs:
                    at = torch.maximum(at, scale[blk])
                    value[blk, :, :lo - j * bs] = _round_code(value[blk, :, :lo - j * bs] / at[:, None, None], kind) * at[:, None, None]
                scale[blk] = at
                value[blk, :, lo - j * bs:hi - j * bs] = _round_code(part / at[:, None, None], kind) * at[:, None, None]
            got = torch.cat([value[b] for b in table[i][:-(-length // bs)]], dim=1)[:, :length]
            back.append(got[:, length - (reads[i + 1] - reads[i]):].transpose(0, 1))
        found[name], found[name + "_scale"] = torch.cat(back), scale
    return found


def _exact_attention(s):
    case = s["case"]
    bs, kv, dim = case["block"], case["kv_heads"], case["dim"]
    group = case["heads"] // kv
    starts, lens = s["q_start"].tolist(), s["lengths"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if case["weights"] else None
    for i, length in enumerate(lens):
        blk = s["table"][i, :-(-length // bs)].long()
        pos = length - (starts[i + 1] - starts[i]) + torch.arange(starts[i + 1] - starts[i], device="cuda")
        j = torch.arange(length, device="cuda")
        hidden = j[None] > pos[:, None]
        if case["window"]:
            hidden |= j[None] <= pos[:, None] - case["window"]
        for h in range(kv):
            k, v = ((s[x][blk, h].double() * s[x + "_scale"][blk, h].double()[:, None, None]).flatten(0, 1)[:length] for x in ("k", "v"))
            for a in range(h * group, (h + 1) * group):
                e = s["q"][starts[i]:starts[i + 1], a].double() @ k.T / math.sqrt(dim)
                e[hidden] = -math.inf
                lse[starts[i]:starts[i + 1], a] = torch.logsumexp(e, 1)
                e = torch.softmax(e, 1)
                out[starts[i]:starts[i + 1], a] = e @ v
                if weights is not None:
                    weights[i, h, :length] += e.sum(0)
    return {"out": out, "lse": lse, **({"weights": weights} if weights is not None else {})}


def _exact_evict(s):
    case = s["case"]
    bs, kind, budget, recent = case["block"], case["codes"], case["budget"], case["recent"]
    lens, table = s["lengths"].tolist(), s["table"].cpu().numpy()
    weights, kept = s["weights"].cpu().numpy(), []
    scales = {n: s[n + "_scale"].double() for n in ("k", "v")}
    back = {"k": [], "v": []}
    left = np.zeros_like(weights, dtype=np.float64)
    for i, length in enumerate(lens):
        count = min(length, budget)
        rows = []
        for h in range(case["kv_heads"]):
            at = np.arange(length)
            if length > budget:
                free = weights[i, h, :length - recent]
                best = np.lexsort((np.arange(free.size), -free))[:budget - recent]
                at = np.concatenate([np.sort(best), np.arange(length - recent, length)])
            left[i, h, :count] = weights[i, h][at]
            rows.append(at)
        at = torch.tensor(np.stack(rows), device="cuda")  # [heads, count]
        h = torch.arange(case["kv_heads"], device="cuda")[:, None]
        blk = torch.tensor(table[i], device="cuda").long()
        for n in ("k", "v"):
            have = s[n + "_scale"].double()[blk[at // bs], h]
            value = s[n].view(torch.int8)[blk[at // bs], h, at % bs].view(s[n].dtype).double() * have[..., None]
            for j in range(-(-count // bs)):
                most = have[:, j * bs:(j + 1) * bs].amax(1)
                scales[n][blk[j]] = most
                part = value[:, j * bs:(j + 1) * bs]
                value[:, j * bs:(j + 1) * bs] = _round_code(part / most[:, None, None], kind) * most[:, None, None]
            back[n].append(value.transpose(0, 1))
    return {"k": torch.cat(back["k"]), "v": torch.cat(back["v"]), "k_scale": scales["k"], "v_scale": scales["v"], "keep": None,
            "lengths": None, "weights": torch.tensor(left, device="cuda")}


def _exact_logits(s):
    case = s["case"]
    x = s["logits"].double()
    for i in range(case["rows"]):
        ids = s["history"][i, :int(s["history_len"][i])].long()
        every = torch.bincount(ids, minlength=case["vocab"]) > 0
        made = torch.bincount(ids[int(s["prompt_len"][i]):], minlength=case["vocab"])
        y, r = x[i], s["repetition"][i].double()
        y = torch.where(every & (y > 0), y / r, torch.where(every, y * r, y))
        y = y - s["frequency"][i].double() * made - s["presence"][i].double() * (made > 0)
        if case["bias"]:
            m = int(s["bias_len"][i])
            y[s["bias_ids"][i, :m].long()] += s["bias_values"][i, :m].double()
        if case["mask"]:
            allowed = np.unpackbits(s["mask"][i].cpu().numpy().view(np.uint8), bitorder="little")[:case["vocab"]]
            y[torch.tensor(allowed == 0, device="cuda")] = -math.inf
        x[i] = y
    return {"logits": x, "best": None}


_EXACT = {"rope": _exact_rope, "append": _exact_append, "attention": _exact_attention, "evict": _exact_evict, "logits": _exact_logits}


def exact(case, seed):
    if case["op"] == "append" and case["batch"] * (case["q_hi"] // case["block"] + 2) > 3000:
        return None  # block by block: too slow
    return _EXACT[case["op"]](prepare(case, seed))
