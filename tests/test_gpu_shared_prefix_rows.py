"""shared_attention over prefixes that few, some and many rows share, in f32
and for the least rows of bf16's kernel, against attention in 64 bits."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import NO_PAGE, Step, stored, upload
from tests.test_gpu_shared_attention import copies, run, share

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 80, 96, 128, 112, 72])
@pytest.mark.parametrize("B,T,heads,kv,tokens,page", [
    (4, 1, 8, 2, 64, 16), (5, 1, 8, 2, 1000, 48), (17, 1, 8, 2, 64, 16), (9, 4, 16, 2, 640, 80), (30, 3, 4, 1, 2048, 64),
    (3, 30, 8, 1, 9000, 256), (33, 1, 2, 1, 17000, 64)])
def test_f32(session, rng, dim, B, T, heads, kv, tokens, page):
    step = copies(rng, B, T, tokens, [(13 * b) % 31 for b in range(B)], heads=heads, kv=kv, dim=dim, page=page,
                  dtype="f32").device(session)
    for scale in (None, -0.1):
        step.check(run(session, step, [tokens], scale=scale), scale=scale)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("B,heads,kv", [(16, 4, 4), (17, 4, 4), (9, 4, 2), (8, 8, 2), (3, 16, 1), (16, 8, 2)])
@pytest.mark.parametrize("tokens", [16, 80, 3000])
def test_few_rows(session, rng, dim, B, heads, kv, tokens):
    step = copies(rng, B, 1, tokens, [(7 * b) % 19 for b in range(B)], heads=heads, kv=kv, dim=dim).device(session)
    step.check(run(session, step, [tokens]))


@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("missing", [[0], [3, 4], [1, 2, 3], [8], list(range(12)), list(range(1, 12, 2))])
@pytest.mark.parametrize("page", [16, 48])
def test_gaps_in_f32(session, rng, dim, missing, page):
    """An odd number of 16-key tiles too, NaNs in the pages that lie behind."""
    step = copies(rng, 20, 1, 12 * page, [3 * b for b in range(20)], heads=8, kv=2, dim=dim, page=page, dtype="f32")
    step.table[:, missing] = NO_PAGE
    step.device(session)
    step.check(run(session, step, [12 * page]))


def test_peaks_that_move_in_f32(session, rng):
    step = copies(rng, 24, 1, 1024, [5] * 24, heads=4, kv=1, dim=80, dtype="f32")
    step.query = stored(np.full((24, 4 * 80), 1.0) + rng.standard_normal((24, 4 * 80)) * 0.1, "f32")
    for n in range(1024):
        _, line = step.place(0, n)
        for b in range(24):
            step.keys[0, step.table[b, n // 16], :, line] = np.float32(n / 64.0)
    step.device(session)
    step.check(run(session, step, [1024]))


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("dim", [64, 80])
def test_committed_values_that_are_not_finite_in_f32(session, rng, value, dim):
    """They reach every row of their key head and dim, and nothing else."""
    step = copies(rng, 20, 1, 256, [2] * 20, heads=8, kv=2, dim=dim, dtype="f32")
    page, line = step.place(0, 100)
    step.values[0, page, 1, line, 7] = value
    step.device(session)
    got = run(session, step, [256]).reshape(20, 8, dim)
    np.testing.assert_array_equal(got[:, 4:, 7], np.full((20, 4), value, np.float32))
    got[:, 4:, 7] = 0
    assert np.isfinite(got).all()


def test_odd_strides_in_f32(session, rng):
    step = copies(rng, 20, 1, 320, [9] * 20, heads=8, kv=2, dim=96, dtype="f32").device(session)
    wide = np.zeros((20, 8 * 96 + 3), np.float32)
    wide[:, 1:-2] = step.query
    query = A.slice(upload(session, wide, "f32"), [{}, {"start": 1, "stop": 8 * 96 + 1}])
    step.check(A.shared_attention(step.cache, step.batch, query, upload(session, np.array([320], np.uint32), "u32")).storage())


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("bf16", 128), ("f32", 64), ("f32", 80)])
@pytest.mark.parametrize("groups,per,T,heads,kv,shared", [
    (1, 70, 3, 4, 2, (400,)), (2, 70, 2, 4, 1, (800, 96)), (3, 9, 5, 8, 1, (64, 1500, 640)), (1, 130, 2, 2, 1, (300,)),
    (2, 40, 4, 2, 2, (0, 333))])
def test_rows_in_use(session, rng, dtype, dim, groups, per, T, heads, kv, shared):
    """Drafts of different lengths, none among them, and sequences that do not hold their group's prefix."""
    B = groups * per
    counts = rng.integers(0, T + 1, B)
    counts[rng.integers(0, B, 3)] = T
    if per > 64:
        counts[:64] = T  # a whole wave of sequences with all their rows, and the rest without
    lengths = np.array([shared[b // per] + (11 * b) % 37 for b in range(B)])
    first = np.arange(groups) * per
    for b in rng.permutation(B)[:B // 6]:
        if b not in first and shared[b // per] > 16:
            lengths[b] = int(rng.integers(0, shared[b // per]))
    step = share(Step(rng, B=B, T=T, heads=heads, kv=kv, dim=dim, lengths=lengths, counts=counts, dtype=dtype, spread=2.0),
                 groups, shared)
    step.query.reshape(B, T, -1)[np.arange(T) >= counts[:, None]] = np.nan if dtype == "f32" else 0x7FC0
    step.device(session)
    got = run(session, step, shared)
    unused = (np.arange(T) >= counts[:, None]).reshape(-1)
    assert not got[unused].any()
    step.check(got, rows=~unused)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_the_first_sequence_does_not_hold_it(session, rng, dtype):
    """Pages are read from the first sequence that does; a group that none does is left to its sequences."""
    step = share(Step(rng, B=60, T=5, heads=2, kv=1, lengths=[200 + b % 7 for b in range(60)], dtype=dtype), 2, [192, 192])
    step.lengths[:5] = 3
    step.lengths[30:] = 100
    step.device(session)
    step.check(run(session, step, [192, 192]))
