"""Drafted tokens over a paged cache: what a decoder block needs between its
quantized projections while T drafted tokens of each of B sequences are
checked at once (T = 1: ordinary decoding; a chain: a piece of a prompt; a
tree: speculative decoding).

* ``PagedCache`` holds the keys and values of one or several layers in pages;
* ``DraftBatch`` says where a step's tokens lie: the page table, how many
  tokens of each sequence are committed, and how many drafted ones are in use;
* ``cache_append`` rotates queries and keys by their positions and appends keys
  and values to a layer;
* ``tree_attention`` attends over the committed tokens and, by a mask, the drafted
  ones;
* ``cache_commit`` keeps the accepted tokens of the draft, in all layers.

Row ``b * T + i`` of an operand is drafted token i of sequence b. All calls
enqueue on the Session's stream and read lengths, tables and masks on the
device, so a captured step is replayed with new ones. Evaluated tensors only:
the cache is written in place, which a Program's nodes are not.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from . import _native
from .core import _ITEMSIZE, _NATIVE_DTYPE, Session, Tensor


_NO_MASK = _native.View()


def _positive(name: str, value: int) -> int:
    if not isinstance(value, int) or isinstance(value, bool) or value <= 0:
        raise TypeError(f"{name} must be a positive integer")
    return value


def _matrix(op: str, name: str, t: Tensor, dtypes: tuple[str, ...], shape: tuple[int | None, int | None]) -> Tensor:
    """A rank-two tensor of one of `dtypes` with consecutive columns; None: any size."""
    if not isinstance(t, Tensor) or len(t.shape) != 2 or t.dtype not in dtypes or \
            any(want is not None and have != want for have, want in zip(t.shape, shape)):
        sizes = ", ".join("*" if s is None else str(s) for s in shape)
        raise TypeError(f"{op} {name} must be a [{sizes}] {'/'.join(dtypes)} tensor")
    if t.shape[1] > 1 and t.strides[1] != 1:
        raise TypeError(f"{op} {name} must have consecutive columns")
    return t


def _words(op: str, name: str, t: Tensor, count: int) -> int:
    """Address of a contiguous rank-one u32 tensor of `count` values."""
    if not isinstance(t, Tensor) or t.dtype != "u32" or t.shape != (count,) or not t.is_contiguous():
        raise TypeError(f"{op} {name} must be a contiguous u32 [{count}] tensor")
    return t.data_ptr


def _output(op: str, out: Tensor | None, session: Session, dtype: str, shape: tuple[int, ...]) -> Tensor:
    if out is None:
        return session.empty(dtype, shape)
    if not isinstance(out, Tensor) or out.session is not session or out.dtype != dtype or out.shape != shape or \
            not out.is_contiguous():
        raise TypeError(f"{op} output must be a contiguous {dtype} {list(shape)} tensor of the same Session")
    return out


def _space(out: Tensor) -> int:
    """Bytes from a tensor's first value to the end of its memory."""
    return out._buffer.nbytes - out.offset * _ITEMSIZE[out.dtype]


class PagedCache:
    """Keys and values ``[layers, pages, kv_heads, page_size, head_dim]`` of one
    Session, f32 or bf16. page_size: a multiple of 16; head_dim: a multiple of
    8, at most 256. Its memory needs no clearing."""

    def __init__(self, session: Session, *, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 dtype: str = "bf16", layers: int = 1):
        self.shape = tuple(_positive(name, value) for name, value in (
            ("layers", layers), ("pages", pages), ("kv_heads", kv_heads), ("page_size", page_size),
            ("head_dim", head_dim)))
        self.layers, self.pages, self.kv_heads, self.page_size, self.head_dim = self.shape
        if dtype not in ("f32", "bf16"):
            raise TypeError("PagedCache requires an f32 or bf16 dtype")
        if page_size % 16:
            raise TypeError("page_size must be a multiple of 16")
        if head_dim % 8 or head_dim > 256:
            raise TypeError("head_dim must be a multiple of 8, at most 256")
        self.session, self.dtype = session, dtype
        self.keys = session.empty(dtype, self.shape)
        self.values = session.empty(dtype, self.shape)
        self._struct = _native.KvCache(self.keys.data_ptr, self.values.data_ptr,
                                       math.prod(self.shape) * _ITEMSIZE[dtype], *self.shape, _NATIVE_DTYPE[dtype])

    def _check(self, op: str, layer: int = 0) -> _native.KvCache:
        self.keys._check_live()
        self.values._check_live()
        if type(layer) is not int or not 0 <= layer < self.layers:
            raise TypeError(f"{op} layer is out of range")
        return self._struct


class DraftBatch:
    """``rows`` drafted tokens of each sequence over a cache. ``page_table``
    u32 [B, columns]: the page of every page_size tokens of a sequence (an
    entry >= pages names none); ``lengths`` u32 [B]: committed tokens;
    ``counts`` u32 [B]: drafted tokens in use (default: all). Drafted token i of
    sequence b is its token lengths[b] + i. The tensors are read when a call
    runs: ``Tensor.write`` puts new values into them for the next step."""

    def __init__(self, page_table: Tensor, lengths: Tensor, rows: int, *, counts: Tensor | None = None):
        _matrix("DraftBatch", "page_table", page_table, ("u32",), (None, None))
        self.sequences, self.rows = page_table.shape[0], _positive("rows", rows)
        self.session = page_table.session
        self.page_table, self.lengths, self.counts = page_table, lengths, counts
        self._struct = _native.DraftBatch(page_table.view(), _words("DraftBatch", "lengths", lengths, self.sequences),
                                          None if counts is None else
                                          _words("DraftBatch", "counts", counts, self.sequences), rows)
        self._tensors = [t for t in (page_table, lengths, counts) if t is not None]
        if any(t.session is not self.session for t in self._tensors):
            raise TypeError("DraftBatch tensors must belong to the same Session")

    def _check(self, op: str, cache: PagedCache, operands: tuple[Tensor | None, ...]) -> _native.DraftBatch:
        for t in self._tensors:
            t._check_live()
        session = self.session
        if cache.session is not session:
            raise TypeError(f"{op} operands must belong to the same Session")
        for t in operands:
            if t is not None and (not isinstance(t, Tensor) or t.session is not session):
                raise TypeError(f"{op} operands must belong to the same Session")
        return self._struct


def rotary_table(session: Session, positions: int, rotary_dim: int, *, theta: float = 10000.0) -> Tensor:
    """f32 [positions, rotary_dim]: the cosines, then the sines, of
    position * theta^(-2j / rotary_dim), computed in 64 bits."""
    _positive("positions", positions)
    if _positive("rotary_dim", rotary_dim) % 2:
        raise TypeError("rotary_dim must be even")
    half = rotary_dim // 2
    angle = np.outer(np.arange(positions), float(theta) ** (-np.arange(half) / half))
    return session.tensor(np.concatenate([np.cos(angle), np.sin(angle)], 1), "f32")


def _query_rows(op: str, cache: PagedCache, batch: DraftBatch, query: Tensor, dtypes: tuple[str, ...]) -> None:
    _matrix(op, "query", query, dtypes, (batch.sequences * batch.rows, None))
    if query.shape[1] % (cache.kv_heads * cache.head_dim):
        raise TypeError(f"{op} query width must be a multiple of kv_heads * head_dim")


# The library checks every operand that reaches it as a view, before it
# enqueues anything. A call whose operands it refuses is explained here, in
# the terms of this module; one that it takes is not checked twice.

def _refused(status: int, op: str, explain) -> None:
    if status == _native.INVALID_SHAPE:
        message = _native.last_error()
        explain()
        raise _native.NativeError(status, f"{op}: {message}")
    _native.check(status, op)


def _rank_two(op: str, name: str, t: Tensor) -> _native.View:
    if len(t.shape) != 2 or t.dtype not in _NATIVE_DTYPE:
        raise TypeError(f"{op} {name} must be a rank-two f32/bf16/u32 tensor")
    return t.view()


def cache_append(cache: PagedCache, batch: DraftBatch, query: Tensor, key: Tensor, value: Tensor,
                 positions: Tensor | None, rotary: Tensor, *, layer: int = 0, interleaved: bool = False,
                 out: Tensor | None = None) -> Tensor:
    """Appends the drafted tokens' keys [B*T, kv_heads*head_dim], rotated by
    their positions, and values to a layer of the cache, and returns the
    rotated queries [B*T, heads*head_dim] in the cache's type. ``positions``
    u32 [B*T] (None: lengths[b] + i); ``rotary``: a ``rotary_table``, whose
    rotary_dim may be less than head_dim; pairs are dims (j, j + rotary_dim/2),
    or neighbours with ``interleaved``. Rows not in use append nothing and
    return zeros. ``out`` may be the query itself, and overlaps no operand
    otherwise."""
    op = "cache_append"
    cache_struct = cache._check(op, layer)
    batch_struct = batch._check(op, cache, (query, key, value, positions, rotary))
    views = _rank_two(op, "query", query), _rank_two(op, "key", key), _rank_two(op, "value", value)
    if rotary.dtype != "f32" or len(rotary.shape) != 2 or not rotary.is_contiguous() or rotary.shape[1] % 2 or \
            not 2 <= rotary.shape[1] <= cache.head_dim:
        raise TypeError("cache_append rotary table must be a contiguous f32 [*, *] tensor, its width even and at most "
                        "head_dim")
    out = _output(op, out, cache.session, cache.dtype, query.shape)
    status = _native.load().affon_rocm_cache_append(
        cache.session._handle, cache_struct, batch_struct,
        _native.AppendDesc(*views, None if positions is None else _words(op, "positions", positions, query.shape[0]),
                           rotary.data_ptr, *rotary.shape, 1 if interleaved else 0, layer, out.data_ptr, _space(out)))
    if status:
        def explain():
            _query_rows(op, cache, batch, query, ("f32", "bf16"))
            for name, t in (("key", key), ("value", value)):
                _matrix(op, name, t, (query.dtype,), (query.shape[0], cache.kv_heads * cache.head_dim))
        _refused(status, op, explain)
    return out


def tree_attention(cache: PagedCache, batch: DraftBatch, query: Tensor, mask: Tensor | None = None, *,
                   layer: int = 0, scale: float | None = None, out: Tensor | None = None) -> Tensor:
    """Attention of drafted tokens' queries [B*T, heads*head_dim] over a layer
    that already holds their keys and values. Row (b, i) sees the lengths[b]
    committed tokens and drafted token j where bit j % 32 of ``mask``[b*T + i,
    j // 32] is set (u32; None: a chain, j <= i). ``scale`` of the scores: by
    default head_dim ** -0.5. A row that sees nothing, or is not in use,
    gives zeros. ``out`` may be the query itself, and overlaps no operand
    otherwise."""
    op = "tree_attention"
    cache_struct = cache._check(op, layer)
    batch_struct = batch._check(op, cache, (query, mask))
    view = _rank_two(op, "query", query)
    out = _output(op, out, cache.session, cache.dtype, query.shape)
    status = _native.load().affon_rocm_tree_attention(
        cache.session._handle, cache_struct, batch_struct,
        _native.AttentionDesc(view, _NO_MASK if mask is None else _rank_two(op, "mask", mask),
                              cache.head_dim ** -0.5 if scale is None else scale, layer, out.data_ptr, _space(out)))
    if status:
        def explain():
            _query_rows(op, cache, batch, query, (cache.dtype,))
            if mask is not None:
                _matrix(op, "mask", mask, ("u32",), (query.shape[0], None))
                if mask.shape[1] * 32 < batch.rows:
                    raise TypeError("tree_attention mask must have a bit for every row of a sequence")
        _refused(status, op, explain)
    return out


def cache_commit(cache: PagedCache, batch: DraftBatch, path: Tensor, accepted: Tensor) -> None:
    """Keeps the accepted tokens of the draft, in every layer: drafted token
    i < accepted[b] of sequence b becomes what drafted token path[b, i] was.
    ``path`` u32 [B, n], n <= rows, ascends strictly along its accepted part;
    ``accepted`` u32 [B]. The caller then adds accepted[b] to lengths[b]."""
    op = "cache_commit"
    cache_struct = cache._check(op)
    batch_struct = batch._check(op, cache, (path, accepted))
    status = _native.load().affon_rocm_cache_commit(cache.session._handle, cache_struct, batch_struct,
                                                    _rank_two(op, "path", path),
                                                    _words(op, "accepted", accepted, batch.sequences))
    if status:
        def explain():
            _matrix(op, "path", path, ("u32",), (batch.sequences, None))
            if path.shape[1] > batch.rows:
                raise TypeError("cache_commit path is longer than the batch's rows")
        _refused(status, op, explain)
