"""A key/value cache in 8 bits (shp_cache8_*): one byte an element, with a scale for each block of
tokens of each KV head.

A serving loop appends the new rows of every sequence, attends to what is cached and, where the
cache has to stay within a budget, adds up the attention weight each token gets and moves the
tokens that matter to another cache.  The reference caches nothing
(source/xla_hlo/tools/run_llama_spirv.py:194-295 recomputes every position).
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np

from ._lib import (Cache8AppendArgs, Cache8AttendArgs, Cache8EvictArgs, Cache8Struct,
                   Cache8WeightsArgs, check, lib)
from .runtime import Context, DeviceTensor

FORMATS = {"i8": 0, "e4m3": 1}


def _ptr(t: Optional[DeviceTensor]):
    return None if t is None else t.ptr


class Cache8:
    """The arrays of a cache and the calls on it.  Arrays that are not given are allocated, and
    freed by close(); their layouts are those of shp_cache8 in include/spirv_hip.h.

    Row tensors ([n_seqs][n][heads][head_dim] unless strides are given as (sequence, row, head),
    in floats) may be padded: counts [n_seqs] says how many of a sequence's n rows are real, and
    row i is token lengths[s] - counts[s] + i.  lengths counts the call's own rows: set_lengths (or
    the caller's own kernel) first, then append and attend.  All calls are asynchronous."""

    def __init__(self, ctx: Context, n_seqs: int, n_kv_heads: int, head_dim: int, capacity: int,
                 block: int = 64, fmt: str = "i8", k: Optional[DeviceTensor] = None,
                 v: Optional[DeviceTensor] = None, k_scale: Optional[DeviceTensor] = None,
                 v_scale: Optional[DeviceTensor] = None,
                 lengths: Optional[DeviceTensor] = None):
        if fmt not in FORMATS:
            raise ValueError(f"format {fmt!r}: one of {', '.join(FORMATS)} is needed")
        if block not in (16, 32, 64, 128):
            raise ValueError(f"blocks of {block} tokens: 16, 32, 64 or 128 are needed")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim {head_dim}: 64 or 128 is needed")
        if n_seqs < 1 or n_kv_heads < 1 or n_seqs * n_kv_heads > 65535:
            raise ValueError(f"{n_seqs} sequences of {n_kv_heads} heads: 1 to 65535 heads of all "
                             "sequences together are needed")
        if not 0 < capacity <= 1 << 22 or capacity % 64 or capacity % block:
            raise ValueError(f"capacity {capacity}: a multiple of 64 and of block is needed, "
                             "4194304 at most")
        self.ctx = ctx
        self.n_seqs, self.n_kv_heads, self.head_dim = n_seqs, n_kv_heads, head_dim
        self.capacity, self.block, self.fmt = capacity, block, fmt
        n = n_seqs * n_kv_heads * capacity
        # the arrays that are given are looked at before any is allocated
        arrays = {"k": (k, n * head_dim, np.uint8), "v": (v, n * head_dim, np.uint8),
                  "k_scale": (k_scale, n // block, np.float32),
                  "v_scale": (v_scale, n // block, np.float32), "lengths": (lengths, n_seqs, np.int32)}
        for t, size, dtype in arrays.values():
            if t is not None and t.nbytes < size * np.dtype(dtype).itemsize:
                raise ValueError(f"an array of {t.nbytes} bytes where the cache needs "
                                 f"{size * np.dtype(dtype).itemsize}")
        self._own = []
        try:
            for name, (t, size, dtype) in arrays.items():
                if t is None:
                    t = DeviceTensor(ctx, size, dtype)
                    self._own.append(t)
                setattr(self, name, t)
            if lengths is None:
                self.lengths.upload(np.zeros(n_seqs, np.int32))
        except BaseException:  # nobody gets an object to close
            for t in self._own:
                t.free()
            raise
        self._struct = Cache8Struct(self.k.ptr, self.v.ptr, self.k_scale.ptr, self.v_scale.ptr,
                                    self.lengths.ptr, n_seqs, n_kv_heads, head_dim, capacity,
                                    block, FORMATS[fmt])
        self._ref = C.byref(self._struct)
        self._lib = lib()
        self._plain = {}  # (rows, heads) -> strides of a tensor without gaps

    def close(self) -> None:
        for t in self._own:
            t.free()
        self._own = []
        # calls on a closed cache are refused
        st = self._struct
        st.k = st.v = st.k_scale = st.v_scale = st.lengths = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def set_lengths(self, lengths: Sequence[int]) -> None:
        """Uploads how many tokens each sequence holds (synchronous)."""
        self.lengths.upload(np.asarray(lengths, np.int32))

    def _strides(self, n: int, heads: int):
        s = self._plain.get((n, heads))
        if s is None:
            d = self.head_dim
            s = self._plain[n, heads] = (n * heads * d, heads * d, d)
        return s

    def append(self, k: DeviceTensor, v: DeviceTensor, n: int,
               counts: Optional[DeviceTensor] = None, k_strides=None, v_strides=None) -> None:
        """Quantises the new rows k and v into the cache (shp_cache8_append)."""
        plain = self._strides(n, self.n_kv_heads)
        args = Cache8AppendArgs(k.ptr, v.ptr, *(k_strides or plain), *(v_strides or plain),
                                _ptr(counts), n)
        rc = self._lib.shp_cache8_append(self.ctx.handle, self._ref, args)
        if rc:
            check(rc, "shp_cache8_append")

    def read(self, n: int, k: Optional[DeviceTensor], v: Optional[DeviceTensor]) -> None:
        """The values of every sequence's newest n tokens, [n_seqs][n_kv_heads][n][head_dim]
        (shp_cache8_read)."""
        rc = self._lib.shp_cache8_read(self.ctx.handle, self._ref, n, _ptr(k), _ptr(v))
        if rc:
            check(rc, "shp_cache8_read")

    def attend(self, q: DeviceTensor, out: DeviceTensor, n_heads: int, n: int,
               counts: Optional[DeviceTensor] = None, lse: Optional[DeviceTensor] = None,
               scale: Optional[float] = None, q_strides=None, o_strides=None) -> None:
        """Attention of n rows a sequence over the cached tokens (shp_cache8_attend); scale is
        head_dim ** -0.5 unless given, lse [n_seqs][n_heads][n] gets the log sums."""
        plain = self._strides(n, n_heads)
        args = Cache8AttendArgs(q.ptr, out.ptr, *(q_strides or plain), *(o_strides or plain),
                                _ptr(counts), _ptr(lse), n, n_heads,
                                self.head_dim ** -0.5 if scale is None else scale)
        rc = self._lib.shp_cache8_attend(self.ctx.handle, self._ref, args)
        if rc:
            check(rc, "shp_cache8_attend")

    def weights(self, q: DeviceTensor, lse: DeviceTensor, acc_in: Optional[DeviceTensor],
                acc_out: DeviceTensor, n_heads: int, n: int,
                counts: Optional[DeviceTensor] = None, scale: Optional[float] = None,
                q_strides=None) -> None:
        """Adds the attention weight that the rows of an attend() gave each token to its account,
        [n_seqs][n_kv_heads][capacity] (shp_cache8_weights)."""
        args = Cache8WeightsArgs(q.ptr, *(q_strides or self._strides(n, n_heads)), _ptr(counts),
                                 lse.ptr, _ptr(acc_in), acc_out.ptr, n, n_heads,
                                 self.head_dim ** -0.5 if scale is None else scale)
        rc = self._lib.shp_cache8_weights(self.ctx.handle, self._ref, args)
        if rc:
            check(rc, "shp_cache8_weights")

    def evict(self, dst: "Cache8", weights: DeviceTensor, keep: int, recent: int,
              kept: DeviceTensor, dst_weights: Optional[DeviceTensor] = None) -> None:
        """Copies each sequence's newest `recent` tokens and the heaviest others, `keep` in all, to
        the cache dst (shp_cache8_evict); kept [n_seqs][n_kv_heads][keep] gets their places."""
        args = Cache8EvictArgs(weights.ptr, kept.ptr, _ptr(dst_weights), keep, recent)
        rc = self._lib.shp_cache8_evict(self.ctx.handle, self._ref, dst._ref, args)
        if rc:
            check(rc, "shp_cache8_evict")
