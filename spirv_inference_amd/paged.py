"""A key/value cache in pages (shp_paged_*): sequences hold tokens in pages that a table hands out, in
fp32, fp16 or bf16.

A serving loop appends the new rows of every sequence, keys and queries turned by their positions on
the way, and attends to what is cached: prompts, single tokens, documents side by side, or trees of
drafted tokens, of which it then keeps the path that the model agrees with.  The reference caches
nothing (source/xla_hlo/tools/run_llama_spirv.py:194-295 recomputes every position).
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Sequence

import numpy as np

from ._lib import (PagedAcceptArgs, PagedAppendArgs, PagedAttendArgs, PagedStruct, check, lib)
from .runtime import Context, DeviceTensor

FORMATS = {"f32": 0, "f16": 1, "bf16": 2}


def _ptr(t: Optional[DeviceTensor]):
    return 0 if t is None else t.ptr


# The arguments' fields in order, as struct writes them into the call's record: a third of the time
# that a new ctypes record takes.
_APPEND = struct.Struct("@2P6q2P6q3P4i")
_ATTEND = struct.Struct("@2P6q6P3i2f")
_ACCEPT = struct.Struct("@8Pi")


class PagedCache:
    """The arrays of a paged cache and the calls on it.  Arrays that are not given are allocated, and
    freed by close(); their layouts are those of shp_paged in include/spirv_hip.h (f16 and bf16 as
    16-bit words).

    Row tensors ([n_seqs][n][heads][head_dim] unless strides are given as (sequence, row, head),
    in floats) may be padded: counts [n_seqs] says how many of a sequence's n rows are real, and
    row i is token lengths[s] - counts[s] + i.  lengths counts the call's own rows: set_lengths (or
    the caller's own kernel) first, then append and attend.  All calls are asynchronous."""

    def __init__(self, ctx: Context, n_seqs: int, n_kv_heads: int, head_dim: int, n_pages: int,
                 page_size: int, max_pages: int, fmt: str = "f32",
                 k: Optional[DeviceTensor] = None, v: Optional[DeviceTensor] = None,
                 table: Optional[DeviceTensor] = None, lengths: Optional[DeviceTensor] = None):
        if fmt not in FORMATS:
            raise ValueError(f"format {fmt!r}: one of {', '.join(FORMATS)} is needed")
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError(f"pages of {page_size} tokens: 16, 32, 64, 128 or 256 are needed")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim {head_dim}: 64 or 128 is needed")
        if n_seqs < 1 or n_kv_heads < 1 or n_seqs * n_kv_heads > 65535:
            raise ValueError(f"{n_seqs} sequences of {n_kv_heads} heads: 1 to 65535 heads of all "
                             "sequences together are needed")
        if n_pages < 1:
            raise ValueError(f"{n_pages} pages: at least one is needed")
        if max_pages < 1 or max_pages * page_size > 1 << 22:
            raise ValueError(f"{max_pages} pages a sequence: 1 to {(1 << 22) // page_size} are needed")
        self.ctx = ctx
        self.n_seqs, self.n_kv_heads, self.head_dim = n_seqs, n_kv_heads, head_dim
        self.n_pages, self.page_size, self.max_pages, self.fmt = n_pages, page_size, max_pages, fmt
        n = n_pages * n_kv_heads * page_size * head_dim
        dtype = np.float32 if fmt == "f32" else np.uint16
        # the arrays that are given are looked at before any is allocated
        arrays = {"k": (k, n, dtype), "v": (v, n, dtype),
                  "table": (table, n_seqs * max_pages, np.int32), "lengths": (lengths, n_seqs, np.int32)}
        for t, size, kind in arrays.values():
            if t is not None and t.nbytes < size * np.dtype(kind).itemsize:
                raise ValueError(f"an array of {t.nbytes} bytes where the cache needs "
                                 f"{size * np.dtype(kind).itemsize}")
        self._own = []
        try:
            for name, (t, size, kind) in arrays.items():
                if t is None:
                    t = DeviceTensor(ctx, size, kind)
                    self._own.append(t)
                setattr(self, name, t)
            if table is None:  # no pages yet
                self.table.upload(np.full(n_seqs * max_pages, -1, np.int32))
            if lengths is None:
                self.lengths.upload(np.zeros(n_seqs, np.int32))
        except BaseException:  # nobody gets an object to close
            for t in self._own:
                t.free()
            raise
        self._struct = PagedStruct(self.k.ptr, self.v.ptr, self.table.ptr, self.lengths.ptr, n_seqs,
                                   n_kv_heads, head_dim, n_pages, page_size, max_pages, FORMATS[fmt])
        self._ref = C.byref(self._struct)
        self._append, self._attend, self._accept = PagedAppendArgs(), PagedAttendArgs(), PagedAcceptArgs()
        self._append_ref, self._attend_ref = C.byref(self._append), C.byref(self._attend)
        self._accept_ref = C.byref(self._accept)
        self._lib = lib()
        self._plain = {}  # (rows, heads) -> strides of a tensor without gaps

    def close(self) -> None:
        for t in self._own:
            t.free()
        self._own = []
        # calls on a closed cache are refused
        st = self._struct
        st.k = st.v = st.table = st.lengths = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def set_lengths(self, lengths: Sequence[int]) -> None:
        """Uploads how many tokens each sequence holds (synchronous)."""
        self.lengths.upload(np.asarray(lengths, np.int32))

    def set_table(self, table) -> None:
        """Uploads the pages of every sequence, [n_seqs][max_pages] (synchronous)."""
        self.table.upload(np.asarray(table, np.int32))

    def _strides(self, n: int, heads: int):
        s = self._plain.get((n, heads))
        if s is None:
            d = self.head_dim
            s = self._plain[n, heads] = (n * heads * d, heads * d, d)
        return s

    def append(self, k: DeviceTensor, v: DeviceTensor, n: int,
               counts: Optional[DeviceTensor] = None, q: Optional[DeviceTensor] = None,
               q_out: Optional[DeviceTensor] = None, n_heads: int = 0,
               inv_freq: Optional[DeviceTensor] = None, rot: Optional[int] = None,
               interleaved: bool = False, offsets: Optional[DeviceTensor] = None, k_strides=None,
               v_strides=None, q_strides=None, o_strides=None) -> None:
        """Stores the new rows k and v, k and q (into q_out) turned by position * inv_freq
        (shp_paged_append); rot is head_dim unless given, or 0 without inv_freq."""
        plain = self._strides(n, self.n_kv_heads)
        heads = self._strides(n, n_heads)
        if rot is None:
            rot = 0 if inv_freq is None else self.head_dim
        _APPEND.pack_into(self._append, 0, k.ptr, v.ptr, *(k_strides or plain),
                          *(v_strides or plain), _ptr(q), _ptr(q_out), *(q_strides or heads),
                          *(o_strides or heads), _ptr(counts), _ptr(offsets), _ptr(inv_freq), n,
                          n_heads, rot, interleaved)
        rc = self._lib.shp_paged_append(self.ctx.handle, self._ref, self._append_ref)
        if rc:
            check(rc, "shp_paged_append")

    def attend(self, q: DeviceTensor, out: DeviceTensor, n_heads: int, n: int,
               counts: Optional[DeviceTensor] = None, lse: Optional[DeviceTensor] = None,
               scale: Optional[float] = None, cap: Optional[float] = None,
               slopes: Optional[DeviceTensor] = None, window: Optional[int] = None,
               prefix: Optional[DeviceTensor] = None, first: Optional[DeviceTensor] = None,
               parents: Optional[DeviceTensor] = None, q_strides=None, o_strides=None) -> None:
        """Attention of n rows a sequence over the cached tokens (shp_paged_attend); scale is
        head_dim ** -0.5 unless given, lse [n_seqs][n_heads][n] gets the log sums."""
        plain = self._strides(n, n_heads)
        _ATTEND.pack_into(self._attend, 0, q.ptr, out.ptr, *(q_strides or plain),
                          *(o_strides or plain), _ptr(counts), _ptr(lse), _ptr(slopes),
                          _ptr(prefix), _ptr(first), _ptr(parents), n, n_heads, window or 0,
                          self.head_dim ** -0.5 if scale is None else scale, cap or 0.0)
        rc = self._lib.shp_paged_attend(self.ctx.handle, self._ref, self._attend_ref)
        if rc:
            check(rc, "shp_paged_attend")

    def accept(self, parents: DeviceTensor, tokens: DeviceTensor, choices: DeviceTensor, n: int,
               path: DeviceTensor, accepted: DeviceTensor, next_ids: DeviceTensor,
               counts: Optional[DeviceTensor] = None,
               lengths_out: Optional[DeviceTensor] = None) -> None:
        """Keeps the path of a drafted tree that the model's choices take (shp_paged_accept);
        lengths_out is the cache's lengths unless given."""
        _ACCEPT.pack_into(self._accept, 0, _ptr(counts), parents.ptr, tokens.ptr, choices.ptr,
                          path.ptr, accepted.ptr, next_ids.ptr,
                          (self.lengths if lengths_out is None else lengths_out).ptr, n)
        rc = self._lib.shp_paged_accept(self.ctx.handle, self._ref, self._accept_ref)
        if rc:
            check(rc, "shp_paged_accept")
