"""Gathered attention weights and eviction by them, against 64 bits."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import NO_PAGE, U, Step, mask_words, set_tensor, tree, upload, widened

pytestmark = pytest.mark.gpu


def gathered(step, mask=None, scale=None, layer=0):
    """(sums [B, kv, capacity] of the probabilities in f64, bound of their error)."""
    capacity = step.table.shape[1] * step.page
    total, bound = (np.zeros((step.B, step.kv, capacity)) for _ in range(2))
    scale = step.dim ** -0.5 if scale is None else scale
    query = widened(step.query).reshape(step.B * step.T, step.heads, step.dim)
    rows = step.T * step.heads // step.kv
    for b in range(step.B):
        keys, _, there = step.tokens(b, layer)
        length, count, n = int(step.lengths[b]), int(step.counts[b]), len(keys)
        for i in range(count):
            seen = there.copy()
            seen[length:] &= (np.arange(count) <= i) if mask is None else mask[b * step.T + i, :count]
            if not seen.any():
                continue
            for h in range(step.heads):
                k = keys[seen, h * step.kv // step.heads]
                s = k @ query[b * step.T + i, h] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                # As of attention: f32 scores, some roundings of the product with the scale, and the sum.
                worst = (np.abs(k) @ np.abs(query[b * step.T + i, h])).max() * abs(scale)
                slack = 2 * (step.dim + 8) * U["f32"] * worst + (len(s) + 16) * U["f32"]
                at = np.nonzero(seen)[0]
                total[b, h * step.kv // step.heads, at] += p
                bound[b, h * step.kv // step.heads, at] += p * (slack + (rows + 4) * U["f32"])
    return total, bound


def check(session, rng, step, mask=None, layer=0, mask_extra=0, **options):
    step.device(session)
    shape = (step.keys.shape[0], step.B, step.kv, step.table.shape[1] * step.page)
    before = rng.uniform(0, 2, shape).astype(np.float32)
    weights = upload(session, before, "f32")
    A.attention_weights(step.cache, step.batch, upload(session, step.query, step.dtype), weights,
                        None if mask is None else upload(session, mask_words(mask, mask_extra), "u32"), layer=layer, **options)
    got = weights.storage()
    total, bound = gathered(step, mask, layer=layer, **options)
    want = before.astype(np.float64)
    n = np.arange(shape[-1])
    for b in range(step.B):
        length, count = int(step.lengths[b]), int(step.counts[b])
        if count == 0:
            continue
        old, new = n < length, (n >= length) & (n < length + count)
        want[layer, b][:, old] += total[b][:, old]
        want[layer, b][:, new] = total[b][:, new]
        size = bound[b] + U["f32"] * np.abs(want[layer, b])
        error = np.abs(got[layer, b] - want[layer, b])
        assert (error <= size)[:, old | new].all(), float((error / np.maximum(size, 1e-300))[:, old | new].max())
        want[layer, b][:, old | new] = got[layer, b][:, old | new]
    np.testing.assert_array_equal(got, want.astype(np.float32))  # the others as they were


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 2), (128, 8, 2), (80, 5, 1), (96, 4, 4), (160, 4, 2), (256, 8, 1), (8, 2, 2),
                                          (200, 3, 3)])
@pytest.mark.parametrize("T,lengths,counts,masked", [
    (1, (0, 1, 15, 16), None, False), (1, (300, 63, 0, 777), (1, 0, 1, 1), False), (5, (14, 100, 3), (5, 0, 3), True),
    (40, (1, 270, 0), (40, 39, 1), True), (33, (70,), None, False)])
def test_sums(session, rng, dtype, dim, heads, kv, T, lengths, counts, masked):
    step = Step(rng, B=len(lengths), T=T, heads=heads, kv=kv, dim=dim, lengths=lengths, counts=counts, dtype=dtype, spread=2.0)
    check(session, rng, step, tree(rng, len(lengths), T) if masked else None, mask_extra=1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,T,length,page", [(1, 1, 5000, 16), (3, 70, 1500, 48), (20, 1, 900, 64), (2, 16, 2100, 32)])
def test_long_contexts(session, rng, dtype, B, T, length, page):
    lengths = [length - 37 * b for b in range(B)]
    check(session, rng, Step(rng, B=B, T=T, heads=8, kv=2, dim=64, page=page, lengths=lengths, dtype=dtype, spread=2.0))


def test_layers_scales_and_gaps(session, rng):
    for layer, scale in ((0, -0.3), (2, 0.0), (1, 1.5)):
        step = Step(rng, B=3, T=4, heads=4, layers=3, lengths=(50, 90, 7), spread=2.0)
        step.table[1, 2] = NO_PAGE
        check(session, rng, step, layer=layer, scale=scale)


def test_rows_that_see_nothing(session, rng):
    """The first token of a sequence whose mask is empty, beside others."""
    step = Step(rng, B=2, T=3, lengths=(0, 0), spread=2.0)
    mask = tree(rng, 2, 3)
    mask[0] = mask[4] = False
    check(session, rng, step, mask)


def test_nans_that_no_row_sees(session, rng):
    """Queries of rows not in use, and what lies in slots of no token: all NaN."""
    step = Step(rng, B=2, T=3, lengths=(30, 31), counts=(2, 3), spread=2.0)
    step.query[2] = 0x7FC0
    check(session, rng, step)


def test_tokens_past_the_table(session, rng):
    step = Step(rng, B=2, T=4, heads=4, lengths=(30, 12), spread=2.0).device(session)
    capacity = step.table.shape[1] * 16
    set_tensor(step.batch.lengths, np.array([capacity - 2, 0xFFFFFFFF], np.uint32))
    step.table[:] = np.arange(step.table.shape[1])
    set_tensor(step.batch.page_table, step.table)
    clean = np.zeros(step.keys.shape, np.uint16)
    set_tensor(step.cache.keys, clean)
    weights = A.token_weights(step.cache, step.batch)
    A.attention_weights(step.cache, step.batch, upload(session, step.query, "bf16"), weights)
    got = weights.numpy()
    # Scores of 0: every seen token gets the same.
    rows = 2  # heads to a key head
    want = np.zeros((2, capacity))
    for i in range(4):
        seen = min(capacity - 2 + i + 1, capacity)
        want[0, :seen] += rows / seen
        want[1] += rows / capacity
    np.testing.assert_allclose(got[0], np.broadcast_to(want[:, None], got[0].shape), rtol=1e-5, atol=0)


def evicted(weights, length, keep, recent):
    """Indices that stay, ascending, of one row of weights."""
    left = min(length, keep)
    recent = min(recent, left)
    others = weights[:length - recent].astype(np.float64)
    others = np.where(np.isnan(others), -np.inf, others)
    nan_last = np.isnan(weights[:length - recent])
    best = np.lexsort((np.arange(len(others)), nan_last, -others))[:left - recent]
    return np.concatenate([np.sort(best), np.arange(length - recent, length)]).astype(int)


def check_evict(session, rng, *, lengths, keep, recent, page=16, dim=64, kv=2, dtype="bf16", layers=2, weights=None,
                in_place=False, gaps=()):
    B = len(lengths)
    step = Step(rng, B=B, T=1, kv=kv, heads=kv, dim=dim, page=page, lengths=lengths, dtype=dtype, layers=layers)
    table = step.table.copy()
    step.device(session)
    capacity = table.shape[1] * page
    before = weights if weights is not None else np.where(rng.random((layers, B, kv, capacity)) < 0.2, 0.0,
                                                          rng.exponential(size=(layers, B, kv, capacity)))
    before = before.astype(np.float32)
    w = upload(session, before, "f32")
    out = A.cache_evict(step.cache, step.batch, w, upload(session, np.array(keep, np.uint32), "u32"),
                        upload(session, np.array(recent, np.uint32), "u32"), out=w if in_place else None)
    if not in_place:
        np.testing.assert_array_equal(w.storage(), before)
    want_w, keys, values = np.zeros_like(before), step.keys.copy(), step.values.copy()
    for layer, b, h in np.ndindex(layers, B, kv):
        length = min(lengths[b], capacity)
        kept = evicted(before[layer, b, h], length, keep[b], recent[b])
        want_w[layer, b, h, :len(kept)] = before[layer, b, h, kept]
        if len(kept) == length:
            continue
        for to, source in enumerate(kept):
            (p, line), (q, from_line) = step.place(b, to), step.place(b, int(source))
            keys[layer, p, h, line] = step.keys[layer, q, h, from_line]
            values[layer, p, h, line] = step.values[layer, q, h, from_line]
    np.testing.assert_array_equal(out.storage(), want_w)
    np.testing.assert_array_equal(step.cache.keys.storage(), keys)
    np.testing.assert_array_equal(step.cache.values.storage(), values)


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("f32", 8), ("bf16", 72), ("bf16", 128), ("f32", 256), ("bf16", 8)])
@pytest.mark.parametrize("lengths,keep,recent,page", [
    ((100, 40, 16, 0), (50, 50, 16, 5), (10, 0, 16, 5), 16), ((700, 1300), (300, 1299), (0, 400), 48),
    ((5, 1, 2), (1, 1, 0), (1, 0, 0), 16), ((64, 65, 63), (63, 64, 1), (63, 1, 9), 64)])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict(session, rng, dtype, dim, lengths, keep, recent, page, in_place):
    check_evict(session, rng, lengths=lengths, keep=keep, recent=recent, page=page, dim=dim, dtype=dtype, in_place=in_place)


def test_evict_long_rows(session, rng):
    """More tokens than a window of the selection, or of the moves, holds."""
    for keep, recent in ((1000, 100), (8000, 4200), (9200, 0)):
        check_evict(session, rng, lengths=(9217, 5000), keep=(keep, 4097), recent=(recent, 3), dim=8, page=64, layers=1)


def test_evict_equal_and_odd_weights(session, rng):
    """Ties go to the first; zeros of both signs are equal; infinities are the most; a NaN is the least."""
    shape = (1, 1, 2, 208)
    for values in ([1.0], [0.0, -0.0], [2.0, 1.0, 1.0], [np.inf, 1.0, -np.inf, np.nan, -0.0, 0.0, 3.5, -2.0], [np.nan],
                   [1.0, np.nextafter(np.float32(1), np.float32(2)), 1e-45, 0.0]):
        weights = rng.choice(np.array(values, np.float32), shape)
        check_evict(session, rng, lengths=(200,), keep=(73,), recent=(11,), layers=1, weights=weights)


def test_evict_again(session, rng):
    """Weights, eviction and the tokens after it, over several rounds: as in a program that keeps
    its cache below a budget."""
    step = Step(rng, B=2, T=4, heads=4, kv=2, lengths=(60, 60), layers=1).device(session)
    set_tensor(step.batch.page_table, step.table)
    weights = A.token_weights(step.cache, step.batch)
    keep, recent = (upload(session, np.array(v, np.uint32), "u32") for v in ([40, 30], [8, 8]))
    state = np.zeros(weights.shape, np.float32)
    for _ in range(3):
        A.attention_weights(step.cache, step.batch, upload(session, step.query, "bf16"), weights)
        step.keys, step.values = step.cache.keys.storage(), step.cache.values.storage()
        total, bound = gathered(step)
        got = weights.storage()
        for b in range(2):
            n = int(step.lengths[b])
            want = total[b][:, :n + 4].copy()
            want[:, :n] += state[0, b, :, :n]
            assert (np.abs(got[0, b, :, :n + 4] - want) <= bound[b][:, :n + 4] + U["f32"] * want).all()
        step.lengths = step.lengths + 4
        set_tensor(step.batch.lengths, step.lengths)
        A.cache_evict(step.cache, step.batch, weights, keep, recent, out=weights)
        want = np.zeros_like(state)
        for b in range(2):
            for h in range(2):
                kept = evicted(got[0, b, h], int(step.lengths[b]), (40, 30)[b], 8)
                want[0, b, h, :len(kept)] = got[0, b, h, kept]
        state = weights.storage()
        np.testing.assert_array_equal(state, want)
        step.lengths = np.array([40, 30], np.uint32)
        set_tensor(step.batch.lengths, step.lengths)
        # The next drafted tokens.
        for b in range(2):
            for i in range(4):
                page, line = step.place(b, int(step.lengths[b]) + i)
                for cache in (step.keys, step.values):
                    cache[0, page, :, line] = rng.integers(0x3F00, 0x3FFF, (2, 64))
        keys, values = step.cache.keys.storage(), step.cache.values.storage()
        for b in range(2):
            for i in range(4):
                page, line = step.place(b, int(step.lengths[b]) + i)
                keys[0, page, :, line], values[0, page, :, line] = step.keys[0, page, :, line], step.values[0, page, :, line]
        set_tensor(step.cache.keys, keys)
        set_tensor(step.cache.values, values)


@pytest.mark.parametrize("T,n", [(1, 1), (9, 5), (40, 23), (40, 40)])
def test_weights_follow_accepted_tokens(session, rng, T, n):
    lengths = (0, 15, 33, 7)
    step = Step(rng, B=4, T=T, lengths=lengths, layers=2).device(session)
    capacity = step.table.shape[1] * 16
    before = rng.uniform(0, 2, (2, 4, 2, capacity)).astype(np.float32)
    weights = upload(session, before, "f32")
    path = np.stack([np.sort(rng.choice(T, n, replace=False)) for _ in lengths]).astype(np.uint32)
    path[1] = np.arange(T - n, T)
    accepted = np.array([n, n, n // 2, 0], np.uint32)
    A.cache_commit(step.cache, step.batch, upload(session, path, "u32"), upload(session, accepted, "u32"), weights=weights)
    want = before.copy()
    for b, length in enumerate(lengths):
        want[:, b, :, length:length + T] = 0.0
        want[:, b, :, length:length + accepted[b]] = before[:, b][:, :, length + path[b, :accepted[b]].astype(int)]
    np.testing.assert_array_equal(weights.storage(), want)
    for got, old in ((step.cache.keys, step.keys), (step.cache.values, step.values)):
        moved = old.copy()
        for b in range(4):
            for i in range(int(accepted[b])):
                page, line = step.place(b, lengths[b] + i)
                source = step.place(b, lengths[b] + int(path[b, i]))
                moved[:, page, :, line] = old[:, source[0], :, source[1]]
        np.testing.assert_array_equal(got.storage(), moved)


def test_weights_commit_beside_the_table(session, rng):
    step = Step(rng, B=3, T=4, lengths=(5, 5, 5)).device(session)
    capacity = step.table.shape[1] * 16
    set_tensor(step.batch.lengths, np.array([5, capacity - 1, 0xFFFFFFFF], np.uint32))
    before = rng.uniform(0, 2, (1, 3, 2, capacity)).astype(np.float32)
    weights = upload(session, before, "f32")
    path = upload(session, np.array([[1, 4, 0xFFFFFFFF], [1, 2, 3], [1, 2, 3]], np.uint32), "u32")
    A.cache_commit(step.cache, step.batch, path, upload(session, np.array([9, 3, 3], np.uint32), "u32"), weights=weights)
    want = before.copy()
    want[0, 0, :, 5] = before[0, 0, :, 6]  # the others of its path name no drafted token, and stay
    want[0, 0, :, 8] = 0.0
    np.testing.assert_array_equal(weights.storage(), want)
