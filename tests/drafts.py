"""Operands of the drafted-token ops and what they compute, in 64 bits."""
from __future__ import annotations

import numpy as np

import affon_amd as A
from oracle import oracle as O

NO_PAGE = 0xFFFFFFFF
U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}  # largest relative error of one rounding


def stored(values, dtype):
    """Storage of f64 values: f32, or bf16 bits."""
    f32 = np.asarray(values, np.float64).astype(np.float32)
    return O.bf16_from_f32(f32) if dtype == "bf16" else f32


def widened(arr):
    return O.f32_from_bf16(arr).astype(np.float64) if arr.dtype == np.uint16 else arr.astype(np.float64)


def upload(session, arr, dtype):
    return session.from_bytes(np.ascontiguousarray(arr), A.TensorSpec(dtype, arr.shape))


def set_tensor(tensor, arr):
    """Writes an array's storage into a contiguous tensor."""
    from affon_amd import _native
    arr = np.ascontiguousarray(arr)
    _native.check(_native.load().affon_rocm_memcpy_h2d(tensor.session._handle, tensor.data_ptr, arr.ctypes.data,
                                                       arr.nbytes), "upload")


class Step:
    """A cache whose slots all hold NaN but the committed and drafted tokens,
    the pages of every sequence scattered, and the batch over it."""

    def __init__(self, rng, *, B=1, T=1, heads=4, kv=2, dim=64, page=16, lengths=(5,), counts=None, dtype="bf16",
                 layers=1, spread=1.0):
        self.B, self.T, self.heads, self.kv, self.dim, self.page, self.dtype = B, T, heads, kv, dim, page, dtype
        self.lengths = np.array(lengths, np.uint32)
        self.counts = np.full(B, T, np.uint32) if counts is None else np.array(counts, np.uint32)
        self.ragged = counts is not None
        need = [(int(n) + T + page - 1) // page for n in self.lengths]
        self.pages = sum(need) + 2
        order = rng.permutation(self.pages)
        self.table = np.full((B, max(need)), NO_PAGE, np.uint32)
        for b in range(B):
            self.table[b, :need[b]] = order[sum(need[:b]):sum(need[:b + 1])]
        shape = (layers, self.pages, kv, page, dim)
        nan = np.full(shape, 0x7FC0, np.uint16) if dtype == "bf16" else np.full(shape, np.nan, np.float32)
        self.keys, self.values = nan.copy(), nan.copy()
        for b in range(B):
            n = int(self.lengths[b] + self.counts[b])
            for cache in (self.keys, self.values):
                cache[:, self.table[b, np.arange(n) // page], :, np.arange(n) % page] = \
                    stored(rng.standard_normal((n, layers, kv, dim)), dtype)
        self.query = stored(rng.standard_normal((B * T, heads * dim)) * spread, dtype)

    def device(self, session):
        self.cache = A.PagedCache(session, layers=self.keys.shape[0], pages=self.pages, kv_heads=self.kv,
                                  page_size=self.page, head_dim=self.dim, dtype=self.dtype)
        set_tensor(self.cache.keys, self.keys)
        set_tensor(self.cache.values, self.values)
        self.batch = A.DraftBatch(upload(session, self.table, "u32"), upload(session, self.lengths, "u32"), self.T,
                                  counts=upload(session, self.counts, "u32") if self.ragged else None)
        return self

    def place(self, b, n):
        return int(self.table[b, n // self.page]), n % self.page

    def tokens(self, b, layer=0):
        """Keys and values of a sequence in f64 [n, kv, dim] and whether each lies anywhere."""
        n = int(self.lengths[b] + self.counts[b])
        page, line = self.table[b, np.arange(n) // self.page].astype(np.int64), np.arange(n) % self.page
        there = page < self.pages
        page = np.where(there, page, 0)
        return widened(self.keys[layer][page, :, line]), widened(self.values[layer][page, :, line]), there

    def attention(self, mask=None, scale=None, layer=0):
        """(output, sum of p |v|, bound of the relative error of p) of every
        row in f64: mask bool [B*T, T], None: a chain. Unseen tokens, whatever
        they hold, take no part."""
        out = np.zeros((self.B * self.T, self.heads, self.dim))
        mass, slack = np.zeros_like(out), np.zeros(out.shape[:2] + (1,))
        scale = self.dim ** -0.5 if scale is None else scale
        query = widened(self.query).reshape(self.B * self.T, self.heads, self.dim)
        for b in range(self.B):
            keys, values, there = self.tokens(b, layer)
            length, count = int(self.lengths[b]), int(self.counts[b])
            for i in range(count):
                r = b * self.T + i
                seen = there.copy()
                seen[length:] &= (np.arange(count) <= i) if mask is None else mask[r, :count]
                if not seen.any():
                    continue
                for h in range(self.heads):
                    k, v = keys[seen, h * self.kv // self.heads], values[seen, h * self.kv // self.heads]
                    s = k @ query[r, h] * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[r, h], mass[r, h] = p @ v, p @ np.abs(v)
                    # f32 scores: the sum's error and some roundings of the product with the scale.
                    worst = (np.abs(k) @ np.abs(query[r, h])).max() * abs(scale)
                    slack[r, h] = 2 * (self.dim + 8) * U["f32"] * worst + (len(s) + 16) * U["f32"]
        return tuple(a.reshape(self.B * self.T, -1) for a in (out, mass, np.broadcast_to(slack, out.shape)))

    def check(self, got, mask=None, scale=None, layer=0, rows=None):
        """got is right: f32 up to the error of f32 sums; bf16 also one rounding
        of the probabilities and one of the result."""
        want, mass, slack = self.attention(mask, scale, layer)
        have = widened(got)
        bound = slack * mass + 1e-30
        if self.dtype == "bf16":
            bound += U["bf16"] * (1 + slack) * (mass + np.abs(want))
        else:
            bound += U["f32"] * np.abs(want)
        rows = slice(None) if rows is None else rows
        error = np.abs(have - want)[rows]
        assert np.isfinite(have[rows]).all()
        assert (error <= bound[rows]).all(), f"off by up to {float((error / bound[rows]).max()):.3g} times the bound"


def tree(rng, B, T, wide=0.5):
    """Random trees: mask bool [B*T, T] of each token's ancestors and itself."""
    mask = np.zeros((B, T, T), bool)
    for b in range(B):
        for i in range(T):
            if i:
                mask[b, i] = mask[b, i - 1 if rng.random() > wide else int(rng.integers(0, i))]
            mask[b, i, i] = True
    return mask.reshape(B * T, T)


def mask_words(mask, extra=0):
    """u32 words of a bool mask, bit j of word j // 32; `extra` more words of ones."""
    rows, T = mask.shape
    padded = np.ones((rows, ((T + 31) // 32 + extra) * 32), np.uint8)
    padded[:, :T] = mask  # the bits past T say nothing
    return np.packbits(padded, axis=1, bitorder="little").view(np.uint32)
