"""The paged cache's writers on the GPU: cache_append against the rotation in
64 bits, cache_commit against a copy of the accepted tokens, bit for bit."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import NO_PAGE, U, Step, set_tensor, stored, upload, widened

pytestmark = pytest.mark.gpu


def rotated(x, angles_c, angles_s, rotary, interleaved):
    """(rows [R, heads, dim] rotated in f64, |x1 c| + |x2 s| and the like: what the f32 error is relative to)."""
    y, size = x.copy(), np.abs(x)
    first = np.arange(0, rotary, 2) if interleaved else np.arange(rotary // 2)
    second = first + (1 if interleaved else rotary // 2)
    c, s = angles_c[:, None], angles_s[:, None]
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    size[..., first] = np.abs(x[..., first] * c) + np.abs(x[..., second] * s)
    size[..., second] = np.abs(x[..., second] * c) + np.abs(x[..., first] * s)
    return y, size


def close(got, want, size, dtype):
    """Three f32 roundings relative to the terms, and one of the result."""
    error = np.abs(widened(got) - want)
    assert (error <= 3 * U["f32"] * size + U[dtype] * (np.abs(want) + 3 * U["f32"] * size)).all(), float(error.max())


@pytest.mark.parametrize("x_dtype,dtype", [("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("dim,rotary,interleaved", [(128, 128, False), (128, 64, True), (80, 40, False), (64, 64, True),
                                                    (72, 10, False), (8, 2, True), (256, 256, False)])
@pytest.mark.parametrize("T,lengths,counts", [(1, (0, 15, 16), None), (5, (14, 100, 3), (5, 0, 3)),
                                              (40, (1, 47, 0), (40, 39, 1))])
def test_append(session, rng, x_dtype, dtype, dim, rotary, interleaved, T, lengths, counts):
    heads, kv, layer, positions = 6, 2, 1, 300
    step = Step(rng, B=3, T=T, heads=heads, kv=kv, dim=dim, lengths=lengths, counts=counts, dtype=dtype,
                layers=3).device(session)
    R = 3 * T
    q, k, v = (stored(rng.standard_normal((R, n * dim)), x_dtype) for n in (heads, kv, kv))
    table = rng.uniform(-1, 1, (positions, rotary)).astype(np.float32)
    place = rng.integers(0, positions, R).astype(np.uint32)
    place[R // 2] = positions + 7  # outside: turned with zeros
    out = A.cache_append(step.cache, step.batch, *(upload(session, t, x_dtype) for t in (q, k, v)),
                         upload(session, place, "u32"), upload(session, table, "f32"), layer=layer,
                         interleaved=interleaved)
    rows = np.where((place < positions)[:, None], table[np.minimum(place, positions - 1)], 0.0).astype(np.float64)
    c, s = rows[:, :rotary // 2], rows[:, rotary // 2:]
    used = np.arange(T)[None, :] < step.counts[:, None]
    want, size = rotated(widened(q).reshape(R, heads, dim), c, s, rotary, interleaved)
    want[~used.reshape(-1)] = size[~used.reshape(-1)] = 0.0
    close(out.storage().reshape(want.shape), want, size, dtype)
    # The other layers, and the slots of no appended token, are as they were.
    got_k, got_v = step.cache.keys.storage(), step.cache.values.storage()
    want_k, size_k = rotated(widened(k).reshape(R, kv, dim), c, s, rotary, interleaved)
    want_v = stored(widened(v), dtype).reshape(R, kv, dim)
    for b in range(3):
        for i in range(int(step.counts[b])):
            page, line = step.place(b, int(step.lengths[b]) + i)
            close(got_k[layer, page, :, line], want_k[b * T + i], size_k[b * T + i], dtype)
            np.testing.assert_array_equal(got_v[layer, page, :, line], want_v[b * T + i])
            got_k[layer, page, :, line], got_v[layer, page, :, line] = (step.keys[layer, page, :, line],
                                                                        step.values[layer, page, :, line])
    np.testing.assert_array_equal(got_k, step.keys)
    np.testing.assert_array_equal(got_v, step.values)


def test_append_positions_by_default_follow_the_lengths(session, rng):
    step = Step(rng, B=2, T=3, lengths=(7, 20)).device(session)
    q, k, v = (upload(session, stored(rng.standard_normal((6, n * 64)), "f32"), "f32") for n in (4, 2, 2))
    table = A.rotary_table(session, 40, 64)
    explicit = upload(session, np.array([7, 8, 9, 20, 21, 22], np.uint32), "u32")
    first = A.cache_append(step.cache, step.batch, q, k, v, explicit, table).storage()
    keys = step.cache.keys.storage()
    np.testing.assert_array_equal(first, A.cache_append(step.cache, step.batch, q, k, v, None, table).storage())
    np.testing.assert_array_equal(keys, step.cache.keys.storage())


def test_rotary_table(session):
    got = A.rotary_table(session, 1000, 32, theta=500000.0).numpy().astype(np.float64)
    angle = np.outer(np.arange(1000), 500000.0 ** (-np.arange(16) / 16))
    np.testing.assert_allclose(got, np.concatenate([np.cos(angle), np.sin(angle)], 1), rtol=0, atol=2.0 ** -24)


def test_append_beside_the_table_and_strided(session, rng):
    """Tokens past the table and on pages that are not there are dropped;
    operands that are columns of one wider tensor, at an odd offset too."""
    for offset in (0, 1):
        step = Step(rng, B=2, T=4, lengths=(14, 30)).device(session)
        step.table[1, 1] = NO_PAGE  # tokens 30, 31 nowhere, 32, 33 on the third page
        set_tensor(step.batch.page_table, step.table)
        wide = rng.standard_normal((8, 8 * 64 + 3)).astype(np.float32)
        whole = upload(session, wide, "f32")
        part = lambda a, b: A.slice(whole, [{}, {"start": offset + a * 64, "stop": offset + b * 64}])
        lengths = np.array([step.table.shape[1] * 16 - 2, 30], np.uint32)
        set_tensor(step.batch.lengths, lengths)
        step.table[0] = np.arange(step.table.shape[1])
        step.table[1, 2] = step.table.shape[1]
        set_tensor(step.batch.page_table, step.table)
        A.cache_append(step.cache, step.batch, part(0, 4), part(4, 6), part(6, 8), None,
                       A.rotary_table(session, 8, 64))
        got = step.cache.values.storage()
        new = stored(wide[:, offset + 6 * 64:offset + 8 * 64], "bf16").reshape(8, 2, 64)
        want = step.values.copy()
        last = step.table[0, -1]
        want[0, last, :, 14], want[0, last, :, 15] = new[0], new[1]
        want[0, step.table[1, 2], :, 0], want[0, step.table[1, 2], :, 1] = new[6], new[7]
        np.testing.assert_array_equal(got, want)
        set_tensor(step.batch.lengths, np.array([0xFFFFFFFF, 0xFFFFFFFE], np.uint32))
        A.cache_append(step.cache, step.batch, part(0, 4), part(4, 6), part(6, 8), None,
                       A.rotary_table(session, 8, 64))
        np.testing.assert_array_equal(step.cache.values.storage(), want)


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f32", 8), ("bf16", 72)])
@pytest.mark.parametrize("T,n", [(1, 1), (9, 5), (40, 23), (40, 40)])
def test_commit(session, rng, dtype, dim, T, n):
    """Paths whose places overlap those they are read from."""
    lengths = (0, 15, 33, 7)
    step = Step(rng, B=4, T=T, dim=dim, lengths=lengths, dtype=dtype, layers=2).device(session)
    path = np.stack([np.sort(rng.choice(T, n, replace=False)) for _ in lengths]).astype(np.uint32)
    path[1] = np.arange(T - n, T)  # the longest overlap
    accepted = np.array([n, n, n // 2, 0], np.uint32)
    A.cache_commit(step.cache, step.batch, upload(session, path, "u32"), upload(session, accepted, "u32"))
    for got, old in ((step.cache.keys, step.keys), (step.cache.values, step.values)):
        want = old.copy()
        for b in range(4):
            for i in range(int(accepted[b])):
                page, line = step.place(b, lengths[b] + i)
                source = step.place(b, lengths[b] + int(path[b, i]))
                want[:, page, :, line] = old[:, source[0], :, source[1]]
        np.testing.assert_array_equal(got.storage(), want)


def test_commit_beside_the_table(session, rng):
    """Paths past the batch's rows, tokens past the table and lengths past it move nothing."""
    step = Step(rng, B=3, T=4, lengths=(5, 5, 5)).device(session)
    set_tensor(step.batch.lengths, np.array([5, step.table.shape[1] * 16 - 1, 0xFFFFFFFF], np.uint32))
    path = upload(session, np.array([[1, 4, 0xFFFFFFFF], [1, 2, 3], [1, 2, 3]], np.uint32), "u32")
    A.cache_commit(step.cache, step.batch, path, upload(session, np.array([9, 3, 3], np.uint32), "u32"))
    want = step.keys.copy()
    want[0, step.table[0, 0], :, 5] = want[0, step.table[0, 0], :, 6]
    np.testing.assert_array_equal(step.cache.keys.storage(), want)
