"""Attention of drafted tokens at every width class and number of rows that a
kernel of its own takes: trees and chains over contexts in one piece and in
several, rows not in use, and a value that is not finite for rows that do not
see it. Against the formula in 64 bits (tests/drafts.py)."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import NO_PAGE, Step, mask_words, set_tensor, stored, tree, upload, widened

pytestmark = pytest.mark.gpu

# Three query heads to a key head: 3 T rows. Up to 16, 32, 64 rows, and more.
T_OF_ROWS = {16: 5, 32: 9, 64: 18, 128: 31}


def attend(session, step, mask=None):
    words = None if mask is None else upload(session, mask_words(mask), "u32")
    return A.tree_attention(step.cache, step.batch, upload(session, step.query, step.dtype), words).storage()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", list(T_OF_ROWS))
@pytest.mark.parametrize("dim", [8, 40, 56, 64, 72, 96, 104, 120, 128, 136, 192, 200, 248, 256])
def test_shapes(session, rng, dim, rows, dtype):
    T, kv = T_OF_ROWS[rows], 2
    step = Step(rng, B=3, T=T, heads=3 * kv, kv=kv, dim=dim, lengths=(60, 700, 0), counts=(T, T - 1, T - 3),
                dtype=dtype, spread=2.0).device(session)
    mask = tree(rng, 3, T, wide=0.9)
    clean = attend(session, step, mask)
    step.check(clean, mask)
    step.check(attend(session, step))
    for b in range(3):
        for row in range(int(step.counts[b]), T):
            assert not clean[b * T + row].any()
    # An infinity in drafted token 1 of each sequence: the rows that do not see it are the same.
    values, column = step.values.copy(), dim - 3
    for b in range(3):
        page, line = step.place(b, int(step.lengths[b]) + 1)
        values[0, page, :, line, column] = stored(np.inf, dtype)
    set_tensor(step.cache.values, values)
    got = attend(session, step, mask)
    sees = np.zeros(3 * T, bool)
    for b in range(3):
        sees[b * T:b * T + int(step.counts[b])] = mask[b * T:b * T + int(step.counts[b]), 1]
    assert sees.any() and not sees.all()
    np.testing.assert_array_equal(got[~sees], clean[~sees])
    seen = widened(got[sees]).reshape(-1, 3 * kv, dim)
    assert np.isposinf(seen[..., column]).all()
    assert np.isfinite(np.delete(seen, column, axis=-1)).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T", [2, 12])
def test_lengths_past_the_table(session, rng, dtype, T):
    """Every token of the table is committed, and no drafted one is seen."""
    step = Step(rng, B=2, T=T, heads=4, kv=2, dim=64, lengths=(64 - T, 64 - T), dtype=dtype).device(session)
    assert step.table.shape[1] * step.page == 64
    for lengths in ((64, 69), (64 + T, 0xFFFFFFFF)):
        set_tensor(step.batch.lengths, np.array(lengths, np.uint32))
        for mask in (None, np.zeros((2 * T, T), bool), np.ones((2 * T, T), bool)):
            # The tokens of the table are those of the step as it was made, drafted ones included.
            step.check(attend(session, step, mask), np.ones((2 * T, T), bool))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,lengths", [(1, (777, 30, 0)), (20, (100, 2000, 5))])
@pytest.mark.parametrize("columns", [600, 8192])
def test_tables_wider_than_the_contexts(session, rng, dtype, T, lengths, columns):
    """Pieces follow the table's width; those past a context's end are empty."""
    step = Step(rng, B=3, T=T, heads=8, kv=2, dim=64, lengths=lengths, dtype=dtype)
    wide = np.full((3, columns), NO_PAGE, np.uint32)
    wide[:, :step.table.shape[1]] = step.table
    wide[:, -1] = 0  # a page that is there, past every context
    step.table = wide
    step.device(session)
    mask = tree(rng, 3, T)
    step.check(attend(session, step, mask), mask)
