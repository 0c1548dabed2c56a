"""Attention over an 8-bit key/value cache: a host-side mirror of the engine's ``j4q_kv_*`` entry points
(include/jax4j_mi355x.h). Engine-local; the reference has no attention.

A decoder step between the projections::

    cache = KvCache(be, layers=32, kv_heads=8, head_dim=128, pages=4096, sequences=64, sequence_pages=512)
    cache.extend([0, 1], [1, 1])                       # a token for each of two sequences
    for layer in range(32):
        be.quant_matvec_into(qkv_weights[layer], x_ptr, 0, qkv_ptr, batch=2)
        cache.append(layer, k_ptr, v_ptr, stride=qkv_rows, rope=rope, q_ptr=qkv_ptr, heads=32, q_stride=qkv_rows)
        cache.attend(layer, qkv_ptr, out_ptr, heads=32, q_stride=qkv_rows)
        be.quant_matvec_into(o_weights[layer], out_ptr, h_ptr, h_ptr, batch=2)

Pointers are device addresses (integers); calls enqueue on ``stream`` (0: the engine stream) and do not wait.
"""
from __future__ import annotations

import ctypes as C
from array import array
from operator import index

import numpy as np

from . import _native as N
from .backend import Mi355xBackend, _addresses, _int32, _int64, check
from .tensor import DType, IllegalArgumentException

def _kind(dtype: DType) -> int:
    if dtype is DType.F32:
        return N.KIND_F32
    if dtype is DType.BF16:
        return N.KIND_BF16
    raise IllegalArgumentException(f"values are F32 or BF16, not {dtype}")


def _ints(values, code="i") -> array:
    """Whole numbers as the library reads them; an array of 64 takes 2 us, where a ctypes one takes 15."""
    try:
        return array(code, values if type(values) is list else list(values))
    except OverflowError:
        raise IllegalArgumentException(f"a number does not fit {8 * array(code).itemsize} bits") from None


def _at(a: array) -> int:
    return a.buffer_info()[0]


def _equal(a, b, what: str) -> None:
    if len(a) != len(b):
        raise IllegalArgumentException(f"{len(a)} sequences, {len(b)} {what}")


class Rope:
    """Rotary positions (``j4q_rope``): tables of cosines and sines [rows, dims / 2], and for every pair of channels the axis
    whose position turns it.

    ``sections``: how many pairs belong to each axis, one axis after another (e.g. time, height, width); ``pair_axis``: the
    axis of each pair instead, in any order. ``positions``: device address of int32 [axes, rows]; 0: a token's place in its
    sequence (``KvCache.append`` alone). ``interleaved``: pair i is channels 2i and 2i + 1, else i and i + dims / 2.
    """

    def __init__(self, cos_ptr: int, sin_ptr: int, rows: int, dims: int, positions: int = 0, sections=None, pair_axis=None,
                 interleaved: bool = False):
        if sections is not None and pair_axis is not None:
            raise IllegalArgumentException("rotary pairs are given their axes by sections or by pair_axis")
        if sections is not None:
            pair_axis = [a for a, n in enumerate(sections) for _ in range(n)]
        axes = None
        if pair_axis is not None:
            axes = [index(a) for a in pair_axis]
            if 2 * len(axes) != dims or any(not 0 <= a < 256 for a in axes):
                raise IllegalArgumentException(f"{len(axes)} pairs with axes of [0, 256), for {dims} rotary channels")
            axes = (C.c_uint8 * len(axes))(*axes)
        self._axes = axes
        cos, sin, at = _addresses(cos_ptr, sin_ptr, positions)
        self.args = N.RopeArgs(cos, sin, _int64(rows), _int32(dims), int(interleaved), at or None, C.cast(axes, C.c_void_p) if axes else None)
        self.ref = C.pointer(self.args)


class KvCache:
    """Paged key/value cache of several sequences in several layers, int8 codes with a scale for every 16 tokens and head."""

    def __init__(self, backend: Mi355xBackend, *, layers: int, kv_heads: int, head_dim: int, pages: int, page_tokens: int = 16,
                 sequences: int = 1, sequence_pages: int | None = None):
        self._be = backend
        self.handle = 0
        sequence_pages = pages if sequence_pages is None else sequence_pages
        self._config = N.KvConfig(*map(_int32, (layers, kv_heads, head_dim, page_tokens)), _int64(pages), *map(_int32, (sequences, sequence_pages)))
        out = C.c_uint64()
        check(backend._lib().j4q_kv_create(C.byref(self._config), C.byref(out)), "kv cache")
        self.handle = out.value

    def destroy(self) -> None:
        """Wait for the device, then free the cache."""
        check(N.load().j4q_kv_destroy(self.handle), "kv destroy")
        self.handle = 0

    def info(self) -> dict:
        d = N.KvDesc()
        check(N.load().j4q_kv_info(self.handle, C.byref(d)), "kv info")
        got = {n: getattr(d, n) for n, _ in N.KvDesc._fields_ if n != "config"}
        return {**{n: getattr(d.config, n) for n, _ in N.KvConfig._fields_}, **got}

    def length(self, seq: int) -> int:
        return int(self.lengths([seq])[0])

    def lengths(self, seqs) -> np.ndarray:
        """Tokens of the sequences, int64 [n]."""
        s = _ints(seqs)
        out = np.empty(len(s), np.int64)
        check(N.load().j4q_kv_tables(self.handle, _at(s), len(s), out.ctypes.data, None, 0), "kv tables")
        return out

    def tables(self, seqs) -> np.ndarray:
        """Pages of the sequences, int32 [n, sequence_pages]; -1: evicted, and behind a sequence's last page."""
        s, width = _ints(seqs), self._config.sequence_pages
        out = np.empty((len(s), width), np.int32)
        check(N.load().j4q_kv_tables(self.handle, _at(s), len(s), None, out.ctypes.data, width), "kv tables")
        return out

    # ---- pages ---------------------------------------------------------------------------
    def extend(self, seqs, tokens, stream: int = 0) -> None:
        """Begin a step: sequence seqs[i] gets tokens[i] more tokens (the step's rows, in this order)."""
        s, t = _ints(seqs), _ints(tokens)
        _equal(s, t, "counts of tokens")
        check(self._be._lib().j4q_kv_extend(self.handle, _at(s), _at(t), len(s), *_addresses(stream)), "kv extend")

    def begin(self, seqs, tokens, stream: int = 0) -> None:
        """Begin a step over the last tokens[i] tokens that sequence seqs[i] has already."""
        s, t = _ints(seqs), _ints(tokens)
        _equal(s, t, "counts of tokens")
        check(self._be._lib().j4q_kv_begin(self.handle, _at(s), _at(t), len(s), *_addresses(stream)), "kv begin")

    def fork(self, src, dst, share: bool = True, stream: int = 0) -> None:
        """The empty sequence dst[i] becomes src[i], sharing its pages or with copies of them."""
        s, d = _ints(src), _ints(dst)
        _equal(s, d, "forks")
        check(self._be._lib().j4q_kv_fork(self.handle, _at(s), _at(d), len(s), int(bool(share)), *_addresses(stream)), "kv fork")

    def truncate(self, seqs, lengths) -> None:
        """Cut sequences to lengths[i] tokens; 0 frees them."""
        s, t = _ints(seqs), _ints(lengths, "q")
        _equal(s, t, "lengths")
        check(self._be._lib().j4q_kv_truncate(self.handle, _at(s), _at(t), len(s)), "kv truncate")

    def evict(self, seqs, window: int, sinks: int = 0, stream: int = 0) -> None:
        """Free the pages that no later token sees through a window of so many tokens and so many first ones."""
        s = _ints(seqs)
        check(self._be._lib().j4q_kv_evict(self.handle, _at(s), len(s), _int32(window), _int32(sinks), *_addresses(stream)), "kv evict")

    def compact(self, stream: int = 0) -> int:
        """Move pages so that those in use are the pool's lowest; how many were moved."""
        n = C.c_int64()
        check(self._be._lib().j4q_kv_compact(self.handle, C.byref(n), *_addresses(stream)), "kv compact")
        return n.value

    # ---- a layer of a step ---------------------------------------------------------------
    def append(self, layer: int, k_ptr: int, v_ptr: int, dtype: DType = DType.F32, *, stride: int = 0, rope: Rope | None = None, q_ptr: int = 0,
               q_out_ptr: int = 0, heads: int = 0, q_stride: int = 0, stream: int = 0) -> None:
        """Store the step's keys and values, [rows, kv_heads, head_dim] each, keys turned by ``rope``; with ``q_ptr`` the
        queries [rows, heads, head_dim] too are turned, into ``q_out_ptr`` (0: in place). Strides are in values, 0: dense."""
        if not type(k_ptr) is type(v_ptr) is type(q_ptr) is type(q_out_ptr) is type(stream) is int:
            k_ptr, v_ptr, q_ptr, q_out_ptr, stream = _addresses(k_ptr, v_ptr, q_ptr, q_out_ptr, stream)
        if stride >> 63 or q_stride >> 63:
            raise IllegalArgumentException(f"strides of {stride}, {q_stride} values")
        a = N.KvAppendArgs(k_ptr, v_ptr, stride, _kind(dtype), _int32(heads), q_ptr, q_out_ptr or q_ptr, q_stride, rope.ref if rope else None)
        check(self._be._lib().j4q_kv_append(self.handle, _int32(layer), C.byref(a), stream), "kv append")

    def attend(self, layer: int, q_ptr: int, out_ptr: int, heads: int, *, q_type: DType = DType.F32, out_type: DType = DType.F32, q_stride: int = 0,
               out_stride: int = 0, window: int = 0, sinks: int = 0, scale: float = 0.0, stream: int = 0) -> None:
        """Attention of the step's queries [rows, heads, head_dim] to the tokens j <= p of their sequence, p their own place,
        with j > p - window (0: no window) or j < sinks. ``scale`` 0: 1 / sqrt(head_dim)."""
        if not type(q_ptr) is type(out_ptr) is type(stream) is int:
            q_ptr, out_ptr, stream = _addresses(q_ptr, out_ptr, stream)
        if q_stride >> 63 or out_stride >> 63:
            raise IllegalArgumentException(f"strides of {q_stride}, {out_stride} values")
        a = N.KvAttendArgs(q_ptr, out_ptr, q_stride, out_stride, _kind(q_type), _kind(out_type), _int32(heads), _int32(window), _int32(sinks), scale)
        check(self._be._lib().j4q_kv_attend(self.handle, _int32(layer), C.byref(a), stream), "kv attend")

    def read(self, layer: int, seqs, first, count: int, k_ptr: int, v_ptr: int, stream: int = 0) -> None:
        """Tokens [first[i], first[i] + count) of seqs[i] as fp32 [n, count, kv_heads, head_dim]; zeros where there is none."""
        s, f = _ints(seqs), _ints(first, "q")
        _equal(s, f, "first tokens")
        k, v, st = _addresses(k_ptr, v_ptr, stream)
        check(self._be._lib().j4q_kv_read(self.handle, _int32(layer), _at(s), _at(f), _int64(count), len(s), k, v, st), "kv read")
