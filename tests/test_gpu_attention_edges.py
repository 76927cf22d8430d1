"""Attention of drafted tokens at scales and scores that are as large as f32 has them."""
import numpy as np
import pytest

from tests.drafts import Step, set_tensor, stored, upload, widened
import affon_amd as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [3.4e38, -3.4e38, 0.0])
def test_scores_of_zero_at_any_scale(session, rng, dtype, scale):
    """Every token weighs the same, however large the scale."""
    step = Step(rng, B=2, T=2, heads=4, kv=2, dim=64, lengths=(70, 3), dtype=dtype)
    step.query[:] = 0
    step.device(session)
    step.check(A.tree_attention(step.cache, step.batch, upload(session, step.query, dtype), scale=scale).storage(),
               scale=scale)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_scores_of_minus_infinity(session, rng, dtype):
    """They weigh nothing, and a row that sees no others gives zeros."""
    step = Step(rng, B=2, T=1, heads=4, kv=2, dim=64, lengths=(0, 40), dtype=dtype).device(session)
    keys = step.keys.copy()
    for b, n in ((0, 0), (1, 7)):
        page, line = step.place(b, n)
        keys[0, page, :, line, 0] = stored(-np.inf, dtype)
    step.query[:] = stored(1.0, dtype)
    set_tensor(step.cache.keys, keys)
    got = A.tree_attention(step.cache, step.batch, upload(session, step.query, dtype)).storage()
    assert not got[0].any()
    # The other sequence as if token 7 lay nowhere: its score is far below the others'.
    page, line = step.place(1, 7)
    step.keys[0, page, :, line] = stored(-1e4, dtype)
    step.check(got, rows=slice(1, 2))
    assert np.isfinite(widened(got)).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim,T", [(64, 1), (128, 1), (128, 5), (80, 7), (112, 1), (128, 12), (128, 30), (256, 3), (256, 20),
                                   (200, 2)])
def test_committed_infinities(session, rng, dtype, dim, T):
    """A committed token's infinity reaches every row in use with its sign, in
    its column only; two of them with other signs, and a NaN, give NaN."""
    step = Step(rng, B=2, T=T, heads=6, kv=2, dim=dim, lengths=(90, 500), counts=(T, max(1, T - 1)),
                dtype=dtype).device(session)
    query = upload(session, step.query, dtype)
    run = lambda: A.tree_attention(step.cache, step.batch, query).storage()
    clean = run()
    step.check(clean)
    used = np.concatenate([np.arange(T) + b * T < b * T + step.counts[b] for b in range(2)])
    for column, entries in enumerate([{3: np.inf}, {40: -np.inf}, {17: np.inf, 31: np.inf}, {5: np.inf, 6: -np.inf},
                                      {88: np.nan}, {0: np.inf, 33: np.inf, 64: -np.inf}]):
        values = step.values.copy()
        for b in range(2):
            for n, value in entries.items():
                page, line = step.place(b, n)
                values[0, page, :, line, column] = stored(value, dtype)
        set_tensor(step.cache.values, values)
        got = run()
        column_of = got.reshape(2 * T, 6, dim)[:, :, column]
        signs = {np.sign(v) for v in entries.values()}
        if len(signs) == 1 and not np.isnan(sum(entries.values())):
            assert (widened(column_of[used]) == signs.pop() * np.inf).all()
        else:
            assert np.isnan(widened(column_of[used])).all()
        assert not got[~used].any()
        column_of[:] = clean.reshape(got.shape[0], 6, dim)[:, :, column]
        step.check(got)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,lengths", [(5, (70, 900)), (40, (0, 1500))])
def test_queries_of_rows_not_in_use(session, rng, dtype, T, lengths):
    """What they hold, NaN included, changes nothing."""
    step = Step(rng, B=2, T=T, heads=4, kv=2, dim=64, lengths=lengths, counts=(T - 2, T - 3), dtype=dtype).device(session)
    run = lambda: A.tree_attention(step.cache, step.batch, upload(session, step.query, dtype)).storage()
    clean = run()
    step.check(clean)
    for bad in (np.nan, np.inf):
        for b, count in enumerate((T - 2, T - 3)):
            step.query[b * T + count:(b + 1) * T] = stored(bad, dtype)
        np.testing.assert_array_equal(run(), clean)
