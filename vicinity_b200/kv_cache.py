"""Key/value cache held in 8 bits, rotary positions, attention and eviction.

The Python side of the cache section of ``include/vicinity_gpu.h``, which
states the semantics.  Tensors are device arrays of PyTorch, or of any library
whose objects have ``data_ptr()``, ``shape``, ``stride()``, ``dtype``,
``is_contiguous()`` and ``device.index`` as PyTorch's, with f32, f16 or bf16
elements; outputs are the caller's.  Work is enqueued on
``stream`` (a cudaStream_t handle, None = the legacy default stream) and the
calls return without waiting for it, so a tensor has to stay alive, and be
ready, in that stream's order.
"""
from __future__ import annotations

import ctypes as C
import math
from array import array

import numpy as np

from . import _lib

_NAMES = {"float32": _lib.F32, "float16": _lib.F16, "bfloat16": _lib.BF16}
_CODES: dict = {}  # by the libraries' own dtype objects, as _TYPES
_TYPES: dict = {}
_SCALINGS = {"none": _lib.ROTARY_PLAIN, "linear": _lib.ROTARY_LINEAR, "by_parts": _lib.ROTARY_BY_PARTS}


def _dtype(x) -> int:
    code = _CODES.get(x.dtype)
    if code is None:
        name = str(x.dtype).rpartition(".")[2]
        if name not in _NAMES:
            raise ValueError(f"tensors are float32, float16 or bfloat16, got {name}")
        code = _CODES[x.dtype] = _NAMES[name]
    return code


def _heads(x, name: str, tokens: int, dim: int, dtype: int) -> tuple:
    """The vg_heads of a [tokens, heads, dim] array with its last dimension contiguous."""
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or shape[0] != tokens or shape[2] != dim:
        raise ValueError(f"{name} must be [{tokens}, heads, {dim}], got {list(shape)}")
    if _CODES.get(x.dtype, -1) != dtype and _dtype(x) != dtype:
        raise ValueError(f"{name} must have the element type of the other tensors")
    if stride[2] != 1 and tokens:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    return x.data_ptr(), shape[1], stride[0], stride[1]


_HEADS = 32  # bytes of a vg_heads


def _flat(x, name: str, shape: tuple, dtype: str) -> int:
    """Address of a contiguous device array of the given shape and type."""
    known = _TYPES.get(x.dtype)
    if known is None:
        known = _TYPES[x.dtype] = str(x.dtype).rpartition(".")[2]
    if known != dtype or x.shape != shape or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} array of shape {list(shape)}")
    return x.data_ptr()


def _any_flat(x, name: str, shape: tuple, dtype: str) -> int:
    """Address of a contiguous host (NumPy) or device array."""
    if isinstance(x, np.ndarray):
        if x.shape != shape or x.dtype != np.dtype(dtype) or not x.flags.c_contiguous:
            raise ValueError(f"{name} must be a contiguous {dtype} array of shape {list(shape)}")
        return x.ctypes.data
    return _flat(x, name, shape, dtype)


class Rotary:
    """Rotary positions: ``layout`` "half" pairs dimension i with i + dim / 2,
    "interleaved" 2i with 2i + 1; ``scaling`` "none", "linear" (frequencies
    divided by ``factor``) or "by_parts" (only those that turn less than
    ``high_turns`` times within ``original_length`` positions, in full below
    ``low_turns``).  ``magnitude`` multiplies every rotated pair."""

    def __init__(self, dim: int, base: float = 10000.0, layout: str = "half", scaling: str = "none",
                 factor: float = 1.0, original_length: float = 0.0, low_turns: float = 1.0,
                 high_turns: float = 32.0, magnitude: float = 1.0):
        if layout not in ("half", "interleaved"):
            raise ValueError('layout must be "half" or "interleaved"')
        if scaling not in _SCALINGS:
            raise ValueError('scaling must be "none", "linear" or "by_parts"')
        if dim < 0:
            raise ValueError("dim must be greater than 0")
        self._h = None
        self._lib = _lib.load()
        p = _lib.VgRotaryParams(dim, int(layout == "interleaved"), _SCALINGS[scaling], base, factor,
                                original_length, low_turns, high_turns, magnitude)
        handle = C.c_void_p()
        _lib.check(self._lib.vg_rotary_create(C.byref(p), C.byref(handle)))
        self._h = handle
        self.dim = dim

    def close(self) -> None:
        if self._h:
            self._lib.vg_rotary_destroy(self._h)
            self._h = None

    def __del__(self):  # pragma: no cover - interpreter shutdown order
        try:
            self.close()
        except Exception:
            pass

    def frequencies(self) -> np.ndarray:
        """Radians per position of the dim / 2 pairs."""
        out = np.empty(self.dim // 2, dtype=np.float64)
        _lib.check(self._lib.vg_rotary_frequencies(self._h, out.ctypes.data))
        return out

    def apply(self, positions, q, k=None, out_q=None, out_k=None, transpose: bool = False, stream=None) -> None:
        """Rotate ``q`` (and ``k``), [tokens, heads, head_dim], at int64
        ``positions`` into ``out_q`` (and ``out_k``); in place without them.
        ``transpose``: the gradient's map."""
        n, d, dt = q.shape[0], q.shape[-1], _dtype(q)
        pos = _flat(positions, "positions", (n,), "int64")
        hq = _heads(q, "q", n, d, dt)
        packed = hq + (hq if out_q is None else _heads(out_q, "out_q", n, d, dt))
        if k is not None:
            hk = _heads(k, "k", n, d, dt)
            packed += hk + (hk if out_k is None else _heads(out_k, "out_k", n, d, dt))
        elif out_k is not None:
            raise ValueError("out_k without k")
        h = array("q", packed)
        at = h.buffer_info()[0]
        _lib.check(self._lib.vg_rotary_apply(
            self._h, dt, d, pos, n, at, at + _HEADS, None if k is None else at + 2 * _HEADS,
            None if k is None else at + 3 * _HEADS, 1 if transpose else 0, q.device.index or 0, stream))


class _Weights:
    """The cache's accumulated weights for libraries that read the CUDA array interface."""

    def __init__(self, cache, ptr, shape, stride):
        self._cache = cache  # keeps the memory alive
        self.__cuda_array_interface__ = {
            "shape": shape,
            "typestr": "<f4",
            "data": (ptr, False),
            "strides": (shape[1] * stride * 4, stride * 4, 4),
            "version": 3,
        }


class KVCache:
    """``num_seqs`` sequences of up to ``capacity`` tokens, each with
    ``num_kv_heads`` keys and values of ``head_dim``, as 8-bit codes with one
    power-of-two scale per head and ``block_tokens`` tokens."""

    def __init__(self, num_seqs: int, capacity: int, num_kv_heads: int, head_dim: int, block_tokens: int = 64,
                 device: int = 0):
        if min(num_seqs, capacity, num_kv_heads, head_dim, block_tokens) < 1:
            raise ValueError("num_seqs, capacity, num_kv_heads, head_dim and block_tokens must be greater than 0")
        self._h = None
        self._lib = _lib.load()
        p = _lib.VgKvParams(num_seqs, capacity, num_kv_heads, head_dim, block_tokens)
        handle = C.c_void_p()
        _lib.check(self._lib.vg_kv_create(C.byref(p), device, C.byref(handle)))
        self._h = handle
        self.num_seqs, self.capacity = int(num_seqs), int(capacity)
        self.num_kv_heads, self.head_dim, self.block_tokens = int(num_kv_heads), int(head_dim), int(block_tokens)
        self.device = device

    def close(self) -> None:
        """Wait for the cache's work and free its memory (views of ``weights`` end with it)."""
        if self._h:
            self._lib.vg_kv_destroy(self._h)
            self._h = None

    def __del__(self):  # pragma: no cover - interpreter shutdown order
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def info(self) -> _lib.VgKvInfo:
        info = _lib.VgKvInfo()
        _lib.check(self._lib.vg_kv_get_info(self._h, C.byref(info)))
        return info

    @property
    def lengths(self) -> np.ndarray:
        """Tokens held by each sequence."""
        out = np.empty(self.num_seqs, dtype=np.uint32)
        _lib.check(self._lib.vg_kv_lengths(self._h, out.ctypes.data))
        return out

    @property
    def weights(self) -> _Weights:
        """Accumulated weights, f32 [num_seqs, num_kv_heads, capacity], in place
        (``torch.as_tensor(cache.weights, device="cuda")``)."""
        ptr = C.c_void_p()
        _lib.check(self._lib.vg_kv_weights(self._h, C.byref(ptr)))
        return _Weights(self, ptr.value, (self.num_seqs, self.num_kv_heads, self.capacity),
                        int(self.info().weight_stride))

    def _counts(self, counts, name: str = "counts"):
        """One unsigned number per sequence: an array, its address and the sum."""
        try:
            c = array("I", counts)
        except (OverflowError, TypeError):
            raise ValueError(f"{name} must not be negative, fractions or above 2^32 - 1") from None
        if len(c) != self.num_seqs:
            raise ValueError(f"{name} must have one entry for each of the {self.num_seqs} sequences")
        return c, c.buffer_info()[0], sum(c)

    def truncate(self, lengths) -> None:
        """Keep the first ``lengths[s]`` tokens of every sequence; 0 empties it.
        A block that is cut keeps its scale."""
        c, ptr, _ = self._counts(lengths, "lengths")
        _lib.check(self._lib.vg_kv_truncate(self._h, ptr))

    def append(self, k, v, counts, stream=None) -> None:
        """Append ``counts[s]`` tokens to every sequence; ``k`` and ``v``
        [sum(counts), num_kv_heads, head_dim] hold them in sequence order."""
        c, ptr, n = self._counts(counts)
        dt = _dtype(k)
        h = array("q", _heads(k, "k", n, self.head_dim, dt) + _heads(v, "v", n, self.head_dim, dt))
        at = h.buffer_info()[0]
        _lib.check(self._lib.vg_kv_append(self._h, ptr, dt, at, at + _HEADS, stream))

    def attend(self, q, counts, out, lse=None, scale: float | None = None, causal: bool = True,
               accumulate: bool = False, stream=None) -> None:
        """Softmax attention of ``counts[s]`` queries per sequence, ``q``
        [sum(counts), heads, head_dim] in f16 or bf16, into ``out`` (and the log
        of the denominators into ``lse``, f32 [sum(counts), heads]).  ``scale``
        defaults to head_dim ** -0.5.  ``accumulate`` adds the probabilities to
        ``weights``.  ``out`` may be ``q``."""
        c, ptr, n = self._counts(counts)
        dt = _dtype(q)
        hq = _heads(q, "q", n, self.head_dim, dt)
        h = array("q", hq + _heads(out, "out", n, self.head_dim, dt))
        at = h.buffer_info()[0]
        _lib.check(self._lib.vg_kv_attend(
            self._h, ptr, dt, at, at + _HEADS, None if lse is None else _flat(lse, "lse", (n, hq[1]), "float32"),
            1.0 / math.sqrt(self.head_dim) if scale is None else scale,
            (_lib.KV_CAUSAL if causal else 0) | (_lib.KV_ACCUMULATE if accumulate else 0), stream))

    def evict(self, src, dst, budget: int, recent: int, kept=None, stream=None) -> None:
        """Cut sequences ``src`` down to ``budget`` tokens each into the
        sequences ``dst``: the ``recent`` newest and those of largest
        accumulated weight.  ``kept``: int32 [len(src), num_kv_heads, budget]."""
        try:
            ids = array("I", src), array("I", dst)
        except (OverflowError, TypeError):
            raise ValueError(f"src and dst must be sequences below {self.num_seqs}") from None
        n = len(ids[0])
        if len(ids[1]) != n:
            raise ValueError("src and dst must have the same length")
        if budget < 1 or recent < 0:
            raise ValueError("budget must be greater than 0 and recent not negative")
        ptr = None if kept is None else _flat(kept, "kept", (n, self.num_kv_heads, budget), "int32") or None
        _lib.check(self._lib.vg_kv_evict(self._h, n, ids[0].buffer_info()[0], ids[1].buffer_info()[0], budget, recent,
                                         ptr, stream))

    def read(self, starts, counts, k, v, stream=None) -> None:
        """The values of tokens [starts[s], starts[s] + counts[s]) of every
        sequence into ``k`` and ``v`` [sum(counts), num_kv_heads, head_dim]
        (exact in bf16 and f32)."""
        first, first_ptr, _ = self._counts(starts, "starts")
        c, ptr, n = self._counts(counts)
        dt = _dtype(k)
        h = array("q", _heads(k, "k", n, self.head_dim, dt) + _heads(v, "v", n, self.head_dim, dt))
        at = h.buffer_info()[0]
        _lib.check(self._lib.vg_kv_read(self._h, first_ptr, ptr, dt, at, at + _HEADS, stream))

    def _shapes(self, n: int):
        h, d, nb = self.num_kv_heads, self.head_dim, -(-n // self.block_tokens)
        return (h, n, d), (h, nb), (h, n)

    def load(self, seq: int, k_codes, k_scales, v_codes, v_scales, weights=None, stream=None) -> None:
        """Set a sequence from host or device arrays as ``export`` returns them
        (weights default to 0).  Scales are powers of two in [2^-100, 2^120] or NaN."""
        n = int(k_codes.shape[1])
        codes, scales, w = self._shapes(n)
        if seq < 0:
            raise ValueError("seq must not be negative")
        _lib.check(self._lib.vg_kv_load(
            self._h, seq, n, _any_flat(k_codes, "k_codes", codes, "int8"),
            _any_flat(k_scales, "k_scales", scales, "float32"), _any_flat(v_codes, "v_codes", codes, "int8"),
            _any_flat(v_scales, "v_scales", scales, "float32"),
            None if weights is None else _any_flat(weights, "weights", w, "float32"), stream))

    def export(self, seq: int, stream=None):
        """(k_codes, k_scales, v_codes, v_scales, weights) of a sequence as NumPy arrays."""
        if not 0 <= seq < self.num_seqs:
            raise ValueError(f"seq must be below {self.num_seqs}")
        codes, scales, w = self._shapes(int(self.lengths[seq]))
        out = (np.empty(codes, np.int8), np.empty(scales, np.float32), np.empty(codes, np.int8),
               np.empty(scales, np.float32), np.empty(w, np.float32))
        _lib.check(self._lib.vg_kv_export(self._h, seq, *[a.ctypes.data for a in out], stream))
        return out
