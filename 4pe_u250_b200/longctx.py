"""Long-context serving operators on torch tensors: the mirror of the
"Long-context serving operators" section of include/i4d.h, through the
binding _i4d_torch.so.

``Context`` inherits ``LongContextOps``, so every operator is a method of a
context.  Tensors live on the context's GPU; the calls run on torch's current
stream of that GPU, allocate their outputs and workspaces through torch (so
they can be captured into a graph) and only enqueue work.
"""
import ctypes
import importlib.machinery
import importlib.util
import os

import numpy as np

ERR_ARG = 1
CODE_INT8, CODE_E4M3 = 0, 1
SCALINGS = {"none": 0, "linear": 1, "base": 2, "parts": 3}

# The C entry points; all but the frequency table are called by _i4d_torch.so.
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


_ops = None


def ops():
    """The torch binding (raises if it was not built; no fallback exists)."""
    global _ops
    if _ops is None:
        import torch  # noqa: F401  (the libraries that the binding needs)
        from . import I4DError, load_library
        load_library()
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_i4d_torch.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: run __graft_entry__.build()")
        loader = importlib.machinery.ExtensionFileLoader("_i4d_torch", path)
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_i4d_torch", loader))
        loader.exec_module(module)
        module.set_error(I4DError)
        _ops = module
    return _ops


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
                       self.block_tokens, self.dim, self.code, self.device_index)

    @classmethod
    def empty(cls, blocks, heads, block_tokens, dim, code="int8", device="cuda"):
        """A cache with zeroed codes and scales."""
        import torch
        kinds = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
        if code not in kinds:
            raise _error(f"code {code!r} is none of {sorted(kinds)}")
        kind = kinds[code]
        k, v = (torch.zeros(blocks, heads, block_tokens, dim, dtype=torch.int8, device=device).view(kind) for _ in range(2))
        return cls(k, v, *(torch.zeros(blocks, heads, device=device) for _ in range(2)))


class LongContextOps:
    """The operators as methods of a context (see include/i4d.h for each)."""

    def _handle(self):
        return self._h.value if self._h else 0

    def ops_check(self):
        """Waits for torch's current stream and raises for what the operators found wrong in device arrays."""
        ops().ops_check(self._handle(), self.device)

    def rope(self, q, k, positions, table, interleaved=True, inverse=False, q_out=None, k_out=None):
        """Rotary positions of q [tokens, heads, dim] and k (or None): (q_out, k_out)."""
        return ops().rope(self._handle(), self.device, q, k, positions, table.turns, table.rot_dim, table.magnitude,
                          interleaved, inverse, q_out, k_out)

    def kv8_append(self, cache, k, v, q_start, lengths, block_table, max_q):
        """Writes new rows k, v [tokens, heads, dim] into the cache; lengths include them."""
        ops().kv8_append(self._handle(), self.device, cache.fields, k, v, q_start, lengths, block_table, max_q)

    def kv8_read(self, cache, q_start, lengths, block_table, max_q, tokens, k_out=None, v_out=None):
        """The last rows of every sequence (q_start counts them) as bfloat16 (k, v) [tokens, heads, dim]."""
        return ops().kv8_read(self._handle(), self.device, cache.fields, q_start, lengths, block_table, max_q, tokens,
                              k_out, v_out)

    def kv8_attention(self, cache, q, q_start, lengths, block_table, max_q, max_length, scale=None, window=0, out=None,
                      lse=None, weights=None, workspace=None):
        """Attention of q [tokens, heads, dim] over the cache (out, of q's type);
        scale defaults to dim^-1/2.  lse: FP32 [tokens, heads] to fill; weights:
        FP32 [batch, cache heads, >= max_length] to which each token's
        probabilities are added."""
        return ops().kv8_attention(self._handle(), self.device, cache.fields, q, q_start, lengths, block_table, max_q,
                                   max_length, scale, window, out, lse, weights, workspace)

    def kv8_evict(self, cache, lengths, block_table, weights, budget, recent, max_length, lengths_out=None, keep=None,
                  weights_out=None, workspace=None):
        """Cuts every sequence to `budget` tokens by accumulated weight, in place:
        (lengths_out, keep, weights_out); weights_out defaults to weights."""
        return ops().kv8_evict(self._handle(), self.device, cache.fields, lengths, block_table, weights, budget, recent,
                               max_length, lengths_out, keep, weights_out, workspace)

    def logits_process(self, logits, out=None, best=None, history=None, history_len=None, prompt_len=None,
                       repetition=None, frequency=None, presence=None, bias_ids=None, bias_values=None, bias_len=None,
                       mask=None):
        """Penalties, biases and a mask on logits [rows, vocab]; best: int32 [rows] to fill."""
        return ops().logits_process(self._handle(), self.device, logits, out, best, history, history_len, prompt_len,
                                    repetition, frequency, presence, bias_ids, bias_values, bias_len, mask)
