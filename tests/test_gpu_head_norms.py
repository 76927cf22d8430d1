"""cache_append with norms of the heads and positions of several axes, against
the formula in 64 bits.

The sum of D squares in f32 is off by at most (D + 2) u of itself, in any
order; the mean, the epsilon, the root, its reciprocal (two ulps each for the
last two) and the two products by which a value gets its norm leave it off by
at most ((D + 4) / 2 + 2 + 2 + 2) u; the rotation adds 3 u of its terms, and the
result is rounded once."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import U, Step, stored, upload, widened

pytestmark = pytest.mark.gpu
EPSILON = 1e-6


def expected(x, weight, cosine, sine, rotary, interleaved):
    """Rows [R, heads, D] normed and turned in f64, and the size of their terms."""
    D = x.shape[-1]
    if weight is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + EPSILON) * weight
    y, size = x.copy(), np.abs(x)
    first = np.arange(0, rotary, 2) if interleaved else np.arange(rotary // 2)
    second = first + (1 if interleaved else rotary // 2)
    c, s = cosine[:, None], sine[:, None]
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    size[..., first] = np.abs(x[..., first] * c) + np.abs(x[..., second] * s)
    size[..., second] = np.abs(x[..., second] * c) + np.abs(x[..., first] * s)
    return y, size * ((D + 4) / 2 + 6 + 3 if weight is not None else 3)


def close(got, want, size, dtype):
    error = np.abs(widened(got) - want)
    bound = U["f32"] * size + U[dtype] * (np.abs(want) + U["f32"] * size)
    assert (error <= bound).all(), float((error / np.maximum(bound, 1e-300)).max())


def check(session, rng, *, T, lengths, counts=None, dim=128, rotary=128, interleaved=False, heads=6, kv=2, x="bf16",
          dtype="bf16", norm="one", weight_dtype="bf16", axes=None, spread=1.0, in_place=False, pad=0, by_default=False):
    B, layer, positions = len(lengths), 1, 300
    step = Step(rng, B=B, T=T, heads=heads, kv=kv, dim=dim, lengths=lengths, counts=counts, dtype=dtype,
                layers=3).device(session)
    R = B * T
    operands, arrays = [], []
    for n in (heads, kv, kv):
        wide = stored(rng.standard_normal((R, n * dim + pad)) * spread, x)
        t = upload(session, wide, x)
        operands.append(A.slice(t, [{}, {"start": pad, "stop": pad + n * dim}]) if pad else t)
        arrays.append(widened(wide)[:, pad:].reshape(R, n, dim))
    weights, norms = [None, None], [None, None]
    for k, n in enumerate((heads, kv)):
        if norm in ("one", "heads") or (norm == "query" and k == 0):
            w = stored(1 + 0.3 * rng.standard_normal(n * dim if norm == "heads" else dim), weight_dtype)
            weights[k], norms[k] = widened(w).reshape(-1, dim), upload(session, w, weight_dtype)
    table = rng.uniform(-1, 1, (positions, rotary)).astype(np.float32)
    count = 1 if axes is None else axes.count
    place = rng.integers(0, positions, (count, R)).astype(np.uint32)
    place[-1, R // 2] = positions + 7  # outside: turned with zeros
    if by_default:
        place[:] = np.minimum((np.array(lengths)[:, None] + np.arange(T)).reshape(-1), 0xFFFFFFFF)
    axis = np.zeros(rotary // 2, int) if axes is None else np.array(axes.axes)
    p = place[axis].T.astype(np.int64)  # [R, pairs]
    inside, pair = p < positions, np.arange(rotary // 2)
    p = np.minimum(p, positions - 1)
    cosine, sine = (np.where(inside, table[p, pair + at], 0.0).astype(np.float64) for at in (0, rotary // 2))
    options = {"out": operands[0]} if in_place else {}
    out = A.cache_append(step.cache, step.batch, *operands,
                         None if by_default else upload(session, place if axes is not None else place[0], "u32"),
                         upload(session, table, "f32"), layer=layer, interleaved=interleaved, query_norm=norms[0],
                         key_norm=norms[1], epsilon=EPSILON, axes=axes, **options)
    want, size = expected(arrays[0], weights[0], cosine, sine, rotary, interleaved)
    used = (np.arange(T)[None, :] < step.counts[:, None]).reshape(-1)
    want[~used] = size[~used] = 0.0
    close(out.storage().reshape(want.shape), want, size, dtype)
    # The other layers, and the slots of no appended token, are as they were.
    got_k, got_v = step.cache.keys.storage(), step.cache.values.storage()
    want_k, size_k = expected(arrays[1], weights[1], cosine, sine, rotary, interleaved)
    want_v = stored(arrays[2], dtype)
    for b in range(B):
        for i in range(int(step.counts[b])):
            page, line = step.place(b, int(step.lengths[b]) + i)
            close(got_k[layer, page, :, line], want_k[b * T + i], size_k[b * T + i], dtype)
            np.testing.assert_array_equal(got_v[layer, page, :, line], want_v[b * T + i])
            got_k[layer, page, :, line], got_v[layer, page, :, line] = (step.keys[layer, page, :, line],
                                                                        step.values[layer, page, :, line])
    np.testing.assert_array_equal(got_k, step.keys)
    np.testing.assert_array_equal(got_v, step.values)


@pytest.mark.parametrize("x,dtype", [("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("dim,rotary,interleaved", [(128, 128, False), (128, 64, True), (80, 40, False), (64, 64, True),
                                                    (72, 10, False), (8, 2, True), (256, 256, False), (248, 246, True)])
@pytest.mark.parametrize("T,lengths,counts", [(1, (0, 15, 16), None), (5, (14, 100, 3), (5, 0, 3)),
                                              (40, (1, 47, 0), (40, 39, 1))])
def test_norms(session, rng, x, dtype, dim, rotary, interleaved, T, lengths, counts):
    check(session, rng, T=T, lengths=lengths, counts=counts, dim=dim, rotary=rotary, interleaved=interleaved, x=x,
          dtype=dtype)


@pytest.mark.parametrize("sections,mixed", [((16, 24, 24), False), ((24, 20, 20), True), ((1, 63), False),
                                            ((16, 16, 16, 16), True), ((64,), False), ((3, 5, 7, 49), False)])
@pytest.mark.parametrize("T,lengths", [(1, (5,)), (33, (0, 100, 7))])
@pytest.mark.parametrize("norm", ["one", None])
def test_axes(session, rng, sections, mixed, T, lengths, norm):
    axes = A.rotary_axes(sections, interleaved=mixed)
    assert [axes.axes.count(a) for a in range(axes.count)] == list(sections)
    for interleaved in (False, True):
        check(session, rng, T=T, lengths=lengths, axes=axes, norm=norm, interleaved=interleaved)


def test_axes_of_each_pair():
    assert A.rotary_axes((2, 3)).axes == (0, 0, 1, 1, 1)
    assert A.rotary_axes((3, 1, 2), interleaved=True).axes == (0, 1, 2, 0, 2, 0)


@pytest.mark.parametrize("changes", [
    {"norm": "heads"}, {"norm": "query"}, {"weight_dtype": "f32"}, {"spread": 1e-4}, {"spread": 1e4}, {"in_place": True},
    {"heads": 2}, {"heads": 34, "kv": 1}, {"by_default": True}, {"x": "f32", "pad": 1}, {"pad": 3, "dim": 80, "rotary": 80},
    {"pad": 4}, {"x": "f32", "dtype": "f32", "in_place": True, "norm": "heads", "weight_dtype": "f32"}])
@pytest.mark.parametrize("T", [2, 35])
def test_operands(session, rng, changes, T):
    check(session, rng, T=T, lengths=(7, 20), **changes)


def test_positions_by_default_on_every_axis(session, rng):
    check(session, rng, T=3, lengths=(7, 20), axes=A.rotary_axes((30, 34)), by_default=True)


def test_axes_on_pairs_of_their_own(session, rng):
    """A pair's axis from any list, and a last axis that no pair has."""
    axes = A.RotaryAxes(int(a) for a in rng.integers(0, 3, 40))
    check(session, rng, T=9, lengths=(3, 90), dim=96, rotary=80, axes=axes)


def test_rows_of_zeros(session, rng):
    check(session, rng, T=3, lengths=(2,), spread=0.0)


def test_without_norms_and_axes_it_is_the_plain_append(session, rng):
    """One axis and no norm through the general form: two products and a sum in
    f32, each rounded or not, are at most 3 u of the terms off on either side."""
    for T in (2, 40):
        step = Step(rng, B=2, T=T, lengths=(7, 20), dtype="f32").device(session)
        q, k, v = (upload(session, stored(rng.standard_normal((2 * T, n * 64)), "f32"), "f32") for n in (4, 2, 2))
        place, table = upload(session, np.arange(2 * T, dtype=np.uint32), "u32"), A.rotary_table(session, 100, 64)
        plain = A.cache_append(step.cache, step.batch, q, k, v, place, table).storage()
        keys = step.cache.keys.storage()
        axes = A.RotaryAxes([0] * 32)
        place = upload(session, np.arange(2 * T, dtype=np.uint32)[None], "u32")
        general = A.cache_append(step.cache, step.batch, q, k, v, place, table, axes=axes).storage()
        np.testing.assert_allclose(general, plain, rtol=0, atol=12 * U["f32"] * np.abs(plain).max())
        np.testing.assert_allclose(step.cache.keys.storage()[~np.isnan(keys)], keys[~np.isnan(keys)], rtol=0,
                                   atol=12 * U["f32"] * np.nanmax(np.abs(keys)))
