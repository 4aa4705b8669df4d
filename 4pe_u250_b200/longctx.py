"""Long-context serving operators on torch tensors: the ctypes mirror of the
"Long-context serving operators" section of include/i4d.h.

``Context`` inherits ``LongContextOps``, so every operator is a method of a
context.  Tensors live on the context's GPU; the calls run on torch's current
stream of that GPU, allocate their outputs and workspaces through torch (so
they can be captured into a graph) and only enqueue work.
"""
import ctypes
import math
import struct

import numpy as np

ERR_ARG = 1
F32, BF16, F16 = 0, 1, 2
CODE_INT8, CODE_E4M3 = 0, 1
SCALINGS = {"none": 0, "linear": 1, "base": 2, "parts": 3}
_LEGACY_STREAM = 1  # cudaStreamLegacy: torch names the legacy default stream 0

# The argument structs of include/i4d.h, in native alignment.
_CACHE = "PPPPiiiii"
_ROPE = struct.Struct("@6P8q8ifP")
_APPEND = struct.Struct("@" + _CACHE + "PP4qPPPq4iP")
_READ = struct.Struct("@" + _CACHE + "PPPPPq3iP")
_ATTENTION = struct.Struct("@" + _CACHE + "PPPP5qPPPq7ifPNP")
_EVICT = struct.Struct("@" + _CACHE + "PPqqPPPPq4iPNP")
_LOGITS = struct.Struct("@13P5q3iP")

SIGNATURES = {
    "i4d_rope_frequencies": [ctypes.c_int, ctypes.c_double, ctypes.c_int, ctypes.c_double, ctypes.c_double,
                             ctypes.c_double, ctypes.c_double, ctypes.c_void_p],
    "i4d_rope": [ctypes.c_void_p, ctypes.c_char_p],
    "i4d_kv8_append": [ctypes.c_void_p, ctypes.c_char_p],
    "i4d_kv8_read": [ctypes.c_void_p, ctypes.c_char_p],
    "i4d_kv8_attention": [ctypes.c_void_p, ctypes.c_char_p],
    "i4d_kv8_attention_workspace": [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p],
    "i4d_kv8_evict": [ctypes.c_void_p, ctypes.c_char_p],
    "i4d_kv8_evict_workspace": [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p],
    "i4d_logits_process": [ctypes.c_void_p, ctypes.c_char_p],
    "i4d_ops_check": [ctypes.c_void_p, ctypes.c_void_p],
}


def _error(message):
    from . import I4DError
    return I4DError(ERR_ARG, message)


def _dtypes():
    import torch
    return {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}


def rope_frequencies(rot_dim, base=10000.0, scaling="none", factor=1.0, original_length=4096, low=1.0, high=32.0):
    """Turns per position in units of 2^-64 (uint64 [rot_dim / 2]) of i4d_rope_frequencies."""
    from . import OK, load_library
    if scaling not in SCALINGS:
        raise _error(f"scaling {scaling!r} is none of {sorted(SCALINGS)}")
    out = np.empty(max(0, rot_dim) // 2, dtype=np.uint64)
    if load_library().i4d_rope_frequencies(rot_dim, base, SCALINGS[scaling], factor, original_length, low, high,
                                           out.ctypes.data) != OK:
        raise _error("i4d_rope_frequencies rejected its arguments")
    return out


class RopeTable:
    """The rotary frequencies of a model on a GPU, and the magnitude that
    cosines and sines are multiplied by.  `scaling`: "none", "linear"
    (frequencies / factor), "base" (a larger base) or "parts" (high frequencies
    kept, low ones divided, a ramp between `low` and `high` turns over
    `original_length`)."""

    def __init__(self, rot_dim, base=10000.0, scaling="none", factor=1.0, original_length=4096, low=1.0, high=32.0,
                 magnitude=1.0, device=None):
        import torch
        turns = rope_frequencies(rot_dim, base, scaling, factor, original_length, low, high)
        self.rot_dim, self.magnitude = rot_dim, float(magnitude)
        self.turns = torch.from_numpy(turns.view(np.int64)).to(device if device is not None else "cuda")


class KV8Cache:
    """A paged cache of 8-bit codes: k, v [blocks, heads, block_tokens, dim]
    int8 or float8_e4m3fn and k_scale, v_scale float32 [blocks, heads], all
    contiguous.  A value is code * scale."""

    def __init__(self, k, v, k_scale, v_scale):
        import torch
        if k.dtype not in (torch.int8, torch.float8_e4m3fn) or v.dtype != k.dtype:
            raise _error("cache codes are int8 or float8_e4m3fn")
        if k.dim() != 4 or v.shape != k.shape or k_scale.shape != k.shape[:2] or v_scale.shape != k.shape[:2]:
            raise _error("cache codes are [blocks, heads, block_tokens, dim], scales [blocks, heads]")
        if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise _error("cache scales are float32")
        parts = (k, v, k_scale, v_scale)
        if not all(x.is_contiguous() and x.device == k.device and x.is_cuda for x in parts):
            raise _error("cache tensors are contiguous and on one GPU")
        self.k, self.v, self.k_scale, self.v_scale = parts
        self.blocks, self.heads, self.block_tokens, self.dim = k.shape
        self.code = CODE_INT8 if k.dtype == torch.int8 else CODE_E4M3
        self.device_index = k.get_device()
        self.fields = (k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), self.blocks, self.heads,
                       self.block_tokens, self.dim, self.code)

    @classmethod
    def empty(cls, blocks, heads, block_tokens, dim, code="int8", device="cuda"):
        """A cache with zeroed codes and scales."""
        import torch
        kind = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}[code]
        k, v = (torch.zeros(blocks, heads, block_tokens, dim, dtype=torch.int8, device=device).view(kind) for _ in range(2))
        return cls(k, v, *(torch.zeros(blocks, heads, device=device) for _ in range(2)))


class LongContextOps:
    """The operators as methods of a context (see include/i4d.h for each)."""

    # -- helpers ------------------------------------------------------------
    def _stream(self):
        import torch
        return torch.cuda.current_stream(self.device).cuda_stream or _LEGACY_STREAM

    def _at(self, t, dtype, what, dims=None):
        """Data pointer of a contiguous-rows tensor of `dtype` on the context's GPU (0 for None)."""
        if t is None:
            return 0
        if t.dtype != dtype:
            raise _error(f"{what} has type {t.dtype}, not {dtype}")
        if t.get_device() != self.device:
            raise _error(f"{what} is not on GPU {self.device}")
        if dims is not None and t.dim() != dims:
            raise _error(f"{what} has {t.dim()} dimensions, not {dims}")
        if t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1:
            raise _error(f"{what} is not contiguous in its last dimension")
        return t.data_ptr()

    def _batch(self, cache, q_start, lengths, block_table):
        import torch
        if cache.device_index != self.device:
            raise _error(f"the cache is not on GPU {self.device}")
        i32 = torch.int32
        at = (self._at(q_start, i32, "q_start", 1), self._at(lengths, i32, "lengths", 1),
              self._at(block_table, i32, "block_table", 2))
        batch = lengths.shape[0]
        if q_start.shape[0] != batch + 1 or block_table.shape[0] != batch:
            raise _error("q_start has batch + 1 entries, lengths and block_table batch")
        if block_table.stride(0) < block_table.shape[1] and batch > 1:
            raise _error("rows of block_table overlap")
        return at, batch, block_table.shape[1] if batch <= 1 else block_table.stride(0)

    def ops_check(self):
        """Waits for torch's current stream and raises for what the operators found wrong in device arrays."""
        self._check(self._L.i4d_ops_check(self._h, self._stream()))

    # -- rotary positions ----------------------------------------------------
    def rope(self, q, k, positions, table, interleaved=True, inverse=False, q_out=None, k_out=None):
        """Rotary positions of q [tokens, heads, dim] and k (or None): (q_out, k_out)."""
        import torch
        code = _dtypes().get(q.dtype)
        if code is None:
            raise _error(f"q has type {q.dtype}")
        tokens, heads, dim = q.shape
        qp = self._at(q, q.dtype, "q", 3)
        kp = self._at(k, q.dtype, "k", 3)
        if k is not None and (k.shape[0] != tokens or k.shape[2] != dim):
            raise _error("k is [tokens, heads, dim] like q")
        pp = self._at(positions, torch.int32, "positions", 1)
        if positions.shape[0] != tokens or (tokens > 1 and positions.stride(0) != 1):
            raise _error("positions is [tokens]")
        tp = self._at(table.turns, torch.int64, "table", 1)
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if k is not None and k_out is None:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        qo = self._at(q_out, q.dtype, "q_out", 3)
        ko = self._at(k_out, q.dtype, "k_out", 3) if k is not None else 0
        if q_out.shape != q.shape or (k is not None and k_out.shape != k.shape):
            raise _error("outputs have the inputs' shapes")
        if k is not None:
            k_heads, ks, kos = k.shape[1], k.stride(), k_out.stride()
        else:
            k_heads, ks, kos = 0, (0, 0), (0, 0)
        qs, qos = q.stride(), q_out.stride()
        args = _ROPE.pack(qp, kp, qo, ko, pp, tp, qs[0], qs[1], ks[0], ks[1], qos[0], qos[1], kos[0], kos[1], tokens,
                          heads, k_heads, dim, table.rot_dim, int(interleaved), int(inverse), code, table.magnitude,
                          self._stream())
        self._check(self._L.i4d_rope(self._h, args))
        return q_out, k_out

    # -- the 8-bit cache ------------------------------------------------------
    def kv8_append(self, cache, k, v, q_start, lengths, block_table, max_q):
        """Writes new rows k, v [tokens, heads, dim] into the cache; lengths include them."""
        code = _dtypes().get(k.dtype)
        if code is None or k.shape != v.shape or k.shape[1:] != (cache.heads, cache.dim):
            raise _error("k and v are [tokens, cache heads, dim] of one type")
        kp, vp = self._at(k, k.dtype, "k", 3), self._at(v, k.dtype, "v", 3)
        at, batch, stride = self._batch(cache, q_start, lengths, block_table)
        args = _APPEND.pack(*cache.fields, kp, vp, k.stride(0), k.stride(1), v.stride(0), v.stride(1), *at, stride,
                            batch, k.shape[0], max_q, code, self._stream())
        self._check(self._L.i4d_kv8_append(self._h, args))

    def kv8_read(self, cache, q_start, lengths, block_table, max_q, tokens, k_out=None, v_out=None):
        """The last rows of every sequence (q_start counts them) as bfloat16 (k, v) [tokens, heads, dim]."""
        import torch
        shape = (tokens, cache.heads, cache.dim)
        if k_out is None:
            k_out = torch.empty(shape, dtype=torch.bfloat16, device=cache.k.device)
        if v_out is None:
            v_out = torch.empty(shape, dtype=torch.bfloat16, device=cache.k.device)
        if k_out.shape != shape or v_out.shape != shape or not (k_out.is_contiguous() and v_out.is_contiguous()):
            raise _error("k_out and v_out are contiguous [tokens, heads, dim]")
        kp, vp = self._at(k_out, torch.bfloat16, "k_out"), self._at(v_out, torch.bfloat16, "v_out")
        at, batch, stride = self._batch(cache, q_start, lengths, block_table)
        args = _READ.pack(*cache.fields, kp, vp, *at, stride, batch, tokens, max_q, self._stream())
        self._check(self._L.i4d_kv8_read(self._h, args))
        return k_out, v_out

    def kv8_attention(self, cache, q, q_start, lengths, block_table, max_q, max_length, scale=None, window=0, out=None,
                      lse=None, weights=None, workspace=None):
        """Attention of q [tokens, heads, dim] over the cache (out, of q's type).
        lse: FP32 [tokens, heads] to fill; weights: FP32 [batch, cache heads,
        >= max_length] to which each token's probabilities are added."""
        import torch
        code = _dtypes().get(q.dtype)
        if code is None:
            raise _error(f"q has type {q.dtype}")
        qp = self._at(q, q.dtype, "q", 3)
        tokens, heads, dim = q.shape
        if dim != cache.dim:
            raise _error(f"q has {dim} values a head, the cache {cache.dim}")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        op = self._at(out, q.dtype, "out", 3)
        if out.shape != q.shape:
            raise _error("out has q's shape")
        lp = self._at(lse, torch.float32, "lse", 2)
        if lse is not None and (lse.shape != (tokens, heads) or not lse.is_contiguous()):
            raise _error("lse is contiguous [tokens, heads]")
        at, batch, stride = self._batch(cache, q_start, lengths, block_table)
        wp, ws = self._at(weights, torch.float32, "weights", 3), 0
        if weights is not None:
            ws = weights.stride(1)
            if weights.shape[:2] != (batch, cache.heads) or weights.shape[2] < max_length or \
                    (batch > 1 and weights.stride(0) != cache.heads * ws):
                raise _error("weights is [batch, cache heads, >= max_length]")
        scale = 1.0 / math.sqrt(dim) if scale is None else scale
        qs, os = q.stride(), out.stride()
        head = (*cache.fields, qp, op, lp, wp, qs[0], qs[1], os[0], os[1], ws, *at, stride, batch, tokens, heads, max_q,
                max_length, window, code, scale)
        space, size = self._workspace(_ATTENTION, self._L.i4d_kv8_attention_workspace, head, workspace, q.device)
        self._check(self._L.i4d_kv8_attention(self._h, _ATTENTION.pack(*head, space, size, self._stream())))
        return out

    def kv8_attention_workspace(self, cache, heads, batch, tokens, max_q, max_length, dtype, weights=False):
        """Bytes of workspace that kv8_attention needs for such a call."""
        code = _dtypes().get(dtype)
        if code is None:
            raise _error(f"no type {dtype}")
        width = -(-max_length // cache.block_tokens)
        fake = cache.k.data_ptr()  # the query reads no array
        head = (*cache.fields, fake, fake, 0, fake if weights else 0, 0, 0, 0, 0, max_length, fake, fake, fake, width,
                batch, tokens, heads, max_q, max_length, 0, code, 1.0)
        need = ctypes.c_size_t(0)
        self._check(self._L.i4d_kv8_attention_workspace(self._h, _ATTENTION.pack(*head, 0, 0, 0), ctypes.byref(need)))
        return need.value

    def _workspace(self, layout, query, head, workspace, device):
        """(pointer, bytes) of the caller's workspace or of a new one of the size needed."""
        import torch
        if workspace is not None:
            return self._at(workspace, torch.uint8, "workspace", 1), workspace.shape[0]
        need = ctypes.c_size_t(0)
        self._check(query(self._h, layout.pack(*head, 0, 0, 0), ctypes.byref(need)))
        if not need.value:
            return 0, 0
        return torch.empty(need.value, dtype=torch.uint8, device=device).data_ptr(), need.value

    def kv8_evict(self, cache, lengths, block_table, weights, budget, recent, max_length, lengths_out=None, keep=None,
                  weights_out=None, workspace=None):
        """Cuts every sequence to `budget` tokens by accumulated weight, in place:
        (lengths_out, keep, weights_out); weights_out defaults to weights."""
        import torch
        i32 = torch.int32
        lp, bp = self._at(lengths, i32, "lengths", 1), self._at(block_table, i32, "block_table", 2)
        batch = lengths.shape[0]
        if cache.device_index != self.device:
            raise _error(f"the cache is not on GPU {self.device}")
        if block_table.shape[0] != batch or (batch > 1 and block_table.stride(0) < block_table.shape[1]):
            raise _error("block_table is [batch, blocks]")
        weights_out = weights if weights_out is None else weights_out
        for name, w in (("weights", weights), ("weights_out", weights_out)):
            self._at(w, torch.float32, name, 3)
            if w.shape[:2] != (batch, cache.heads) or w.shape[2] < max_length or \
                    (batch > 1 and w.stride(0) != cache.heads * w.stride(1)):
                raise _error(f"{name} is [batch, cache heads, >= max_length]")
        if lengths_out is None:
            lengths_out = torch.empty_like(lengths)
        if keep is None:
            keep = torch.empty(batch, cache.heads, budget, dtype=i32, device=lengths.device)
        op, kp = self._at(lengths_out, i32, "lengths_out", 1), self._at(keep, i32, "keep", 3)
        if lengths_out.shape != lengths.shape or keep.shape != (batch, cache.heads, budget) or not keep.is_contiguous():
            raise _error("lengths_out is [batch], keep contiguous [batch, cache heads, budget]")
        stride = block_table.shape[1] if batch <= 1 else block_table.stride(0)
        head = (*cache.fields, weights.data_ptr(), weights_out.data_ptr(), weights.stride(1), weights_out.stride(1), lp,
                op, kp, bp, stride, batch, budget, recent, max_length)
        space, size = self._workspace(_EVICT, self._L.i4d_kv8_evict_workspace, head, workspace, lengths.device)
        self._check(self._L.i4d_kv8_evict(self._h, _EVICT.pack(*head, space, size, self._stream())))
        return lengths_out, keep, weights_out

    # -- logits ----------------------------------------------------------------
    def logits_process(self, logits, out=None, best=None, history=None, history_len=None, prompt_len=None,
                       repetition=None, frequency=None, presence=None, bias_ids=None, bias_values=None, bias_len=None,
                       mask=None):
        """Penalties, biases and a mask on logits [rows, vocab]; best: int32 [rows] to fill."""
        import torch
        code = _dtypes().get(logits.dtype)
        if code is None:
            raise _error(f"logits have type {logits.dtype}")
        i32, f32 = torch.int32, torch.float32
        xp = self._at(logits, logits.dtype, "logits", 2)
        rows, vocab = logits.shape
        if out is None:
            out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        op = self._at(out, logits.dtype, "out", 2)
        if out.shape != logits.shape:
            raise _error("out has the logits' shape")
        per_row = [self._at(t, d, n, 1) for t, d, n in (
            (best, i32, "best"), (history_len, i32, "history_len"), (prompt_len, i32, "prompt_len"),
            (repetition, f32, "repetition"), (frequency, f32, "frequency"), (presence, f32, "presence"),
            (bias_len, i32, "bias_len"))]
        for t in (best, history_len, prompt_len, repetition, frequency, presence, bias_len):
            if t is not None and t.shape[0] != rows:
                raise _error("per-row arrays have one entry a row")
        table = [self._at(t, d, n, 2) for t, d, n in ((history, i32, "history"), (bias_ids, i32, "bias_ids"),
                                                      (bias_values, f32, "bias_values"), (mask, i32, "mask"))]
        strides = []
        for t in (history, bias_ids, mask):
            if t is not None and t.shape[0] != rows:
                raise _error("history, biases and mask have one row a row of logits")
            strides.append(0 if t is None else t.shape[1] if rows == 1 else t.stride(0))
        if history is not None and strides[0] < history.shape[1] or bias_ids is not None and strides[1] < bias_ids.shape[1]:
            raise _error("rows of history or biases overlap")
        if bias_ids is not None and (bias_values is None or bias_values.shape != bias_ids.shape or
                                     (rows > 1 and bias_values.stride(0) != strides[1])):
            raise _error("bias_values has bias_ids' shape and strides")
        if mask is not None and mask.shape[1] * 32 < vocab:
            raise _error("mask has fewer than vocab bits a row")
        args = _LOGITS.pack(xp, op, per_row[0], table[0], per_row[1], per_row[2], per_row[3], per_row[4], per_row[5],
                            table[1], table[2], per_row[6], table[3], logits.stride(0), out.stride(0), *strides, rows,
                            vocab, code, self._stream())
        self._check(self._L.i4d_logits_process(self._h, args))
        return out
