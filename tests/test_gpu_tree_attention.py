"""Attention of drafted tokens over a paged cache, on the GPU, against the
formula in 64 bits (tests/drafts.py, which also derives the bound of the
error). Every slot of the cache that no row sees holds NaN."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import NO_PAGE, Step, mask_words, set_tensor, stored, tree, upload, widened
from tests.helpers import HipRuntime

pytestmark = pytest.mark.gpu


def attend(session, step, mask=None, **options):
    words = None if mask is None else upload(session, mask_words(mask), "u32")
    query = upload(session, step.query, step.dtype)
    return A.tree_attention(step.cache, step.batch, query, words, **options).storage()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 4), (128, 8, 2), (80, 5, 1), (8, 2, 2), (256, 6, 2), (104, 9, 3),
                                          (128, 24, 1)])
@pytest.mark.parametrize("T,lengths", [(1, (0, 1, 33)), (3, (16, 31, 0)), (17, (200, 15, 47))])
def test_trees(session, rng, dtype, dim, heads, kv, T, lengths):
    step = Step(rng, B=3, T=T, heads=heads, kv=kv, dim=dim, lengths=lengths, dtype=dtype, spread=2.0).device(session)
    mask = tree(rng, 3, T)
    step.check(attend(session, step, mask), mask)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,length", [(1, 1), (2, 0), (33, 7), (65, 100), (130, 0), (300, 40)])
def test_chains(session, rng, dtype, T, length):
    """No mask: a prompt's piece of any length."""
    step = Step(rng, T=T, heads=4, kv=2, dim=64, lengths=(length,), dtype=dtype).device(session)
    step.check(attend(session, step))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,heads,kv,lengths", [(1, 8, 1, (5000,)), (1, 32, 8, (700, 4095, 2, 1500)),
                                                (24, 16, 2, (3001, 15)), (70, 16, 2, (2050, 333))])
def test_long_contexts(session, rng, dtype, T, heads, kv, lengths):
    """Contexts that are cut into pieces whose results are joined."""
    step = Step(rng, B=len(lengths), T=T, heads=heads, kv=kv, dim=128, lengths=lengths, dtype=dtype,
                spread=3.0).device(session)
    mask = tree(rng, len(lengths), T)
    got = attend(session, step, mask)
    step.check(got, mask)
    np.testing.assert_array_equal(got, attend(session, step, mask))  # the order of the sums is fixed


@pytest.mark.parametrize("page", [16, 48, 64, 80, 256])
def test_pages(session, rng, page):
    """Page sizes that are no power of two, and pages that end inside a tile."""
    step = Step(rng, B=2, T=9, heads=8, kv=2, dim=128, page=page, lengths=(page * 3 - 4, 77)).device(session)
    mask = tree(rng, 2, 9)
    step.check(attend(session, step, mask), mask)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_not_in_use_and_rows_that_see_nothing(session, rng, dtype):
    step = Step(rng, B=4, T=6, heads=8, kv=2, dim=64, lengths=(40, 0, 0, 130), counts=(4, 3, 0, 6),
                dtype=dtype).device(session)
    mask = tree(rng, 4, 6)
    mask[6:9] = False  # sequence 1 has nothing before its drafts
    mask[18:24] = False  # sequence 3 has
    got = attend(session, step, mask)
    step.check(got, mask)
    for r in (4, 5, 6, 7, 8, 9, 12, 17):
        assert not got[r].any(), r


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,length", [(5, 3), (40, 90)])
def test_masked_infinities_and_nan_stay_out(session, rng, dtype, T, length):
    """Rows that do not see a drafted token are the same whatever its key and
    value hold; rows that see it are not finite."""
    step = Step(rng, T=T, heads=8, kv=2, dim=64, lengths=(length,), dtype=dtype).device(session)
    mask = tree(rng, 1, T, wide=0.9)
    clean = attend(session, step, mask)
    step.check(clean, mask)
    for bad, (key, value) in enumerate([(np.nan, np.nan), (1.0, np.inf), (1.0, -np.inf), (np.inf, 1.0), (1.0, np.nan)]):
        j = 1 + bad % (T - 1)
        page, line = step.place(0, length + j)
        keys, values = step.keys.copy(), step.values.copy()
        keys[0, page, :, line], values[0, page, :, line] = stored(key, dtype), stored(value, dtype)
        set_tensor(step.cache.keys, keys)
        set_tensor(step.cache.values, values)
        got = attend(session, step, mask)
        blind = ~mask[:, j]
        step.check(got, mask, rows=blind)
        np.testing.assert_array_equal(got[blind], clean[blind])
        assert blind.sum() and not blind.all()
        if key == 1.0:  # a seen infinity or NaN is what the sum says
            from tests.drafts import widened
            assert not np.isfinite(widened(got[~blind])).any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [24, 72, 80, 96, 112, 160, 192])
@pytest.mark.parametrize("T", [5, 21])
def test_odd_widths(session, rng, T, dtype, dim):
    """Heads whose rows lie in the banks in other orders: trees over a few
    steps, and a value that is not finite for the rows that do not see it."""
    step = Step(rng, T=T, heads=6, kv=2, dim=dim, lengths=(75,), dtype=dtype, spread=2.0).device(session)
    mask = tree(rng, 1, T, wide=0.9)
    clean = attend(session, step, mask)
    step.check(clean, mask)
    for j in range(1, T, 3):
        blind = ~mask[:, j]
        page, line = step.place(0, 75 + j)
        values = step.values.copy()
        values[0, page, :, line, j] = stored(np.inf, dtype)
        set_tensor(step.cache.values, values)
        got = attend(session, step, mask)
        assert blind.any()
        np.testing.assert_array_equal(got[blind], clean[blind])
        seen = widened(got[~blind]).reshape(-1, 6, dim)
        assert np.isposinf(seen[..., j]).all()
        assert np.isfinite(np.delete(seen, j, axis=-1)).all()


def test_scores_far_apart(session, rng):
    """The running maximum: scores to +-3000, the largest early, late and between."""
    for dtype in ("bf16", "f32"):
        for where in (0, 37, 399):
            step = Step(rng, T=1, heads=4, kv=1, dim=64, lengths=(400,), dtype=dtype, spread=100.0).device(session)
            page, line = step.place(0, where)
            step.keys[0, page, :, line] = stored(np.sign(rng.standard_normal((1, 64))) * 4, dtype)
            set_tensor(step.cache.keys, step.keys)
            step.check(attend(session, step, scale=0.2), scale=0.2)


def test_pages_that_are_not_there(session, rng):
    """A table entry that names no page hides its tokens; lengths past the
    table are cut to it."""
    step = Step(rng, B=2, T=2, heads=4, kv=2, dim=64, lengths=(70, 70)).device(session)
    step.table[0, 1] = NO_PAGE
    step.table[1, 3] = step.pages
    set_tensor(step.batch.page_table, step.table)
    step.check(attend(session, step))
    # The whole table of both sequences is committed, and the drafts lie past it.
    capacity = step.table.shape[1] * step.page
    set_tensor(step.batch.lengths, np.array([capacity + 5, 0xFFFFFFFF], np.uint32))
    attend(session, step)  # tokens there hold NaN; nothing past the table is read


def test_strided_and_unaligned_operands(session, rng):
    """Queries that are columns of a wider tensor, at odd offsets; masks and
    tables with longer rows; an output inside a larger buffer."""
    for dtype in ("bf16", "f32"):
        step = Step(rng, B=2, T=5, heads=4, kv=2, dim=64, lengths=(30, 99), dtype=dtype)
        wide = np.full((2, step.table.shape[1] + 3), NO_PAGE, np.uint32)
        wide[:, 1:-2] = step.table
        step.device(session)
        table = A.slice(upload(session, wide, "u32"), [{}, {"start": 1, "stop": wide.shape[1] - 2}])
        batch = A.DraftBatch(table, step.batch.lengths, 5)
        mask = tree(rng, 2, 5)
        words = A.slice(upload(session, np.repeat(mask_words(mask), 3, axis=1), "u32"), [{}, {"start": 2}])
        for offset in (1, 8, 0):
            padded = np.zeros((10, 4 * 64 + 11), step.query.dtype)
            padded[:, offset:offset + 256] = step.query
            query = A.slice(upload(session, padded, dtype), [{}, {"start": offset, "stop": offset + 256}])
            whole = session.empty(dtype, (12, 256))
            out = A.slice(whole, [{"start": 1, "stop": 11}, {}])
            got = A.tree_attention(step.cache, batch, query, words, out=out).storage()
            step.check(got, mask)


def test_layers_and_offsets_past_32_bits(session, rng):
    """A cache of more than 4 GiB of keys, its tokens at the end."""
    step = Step(rng, T=3, heads=8, kv=8, dim=128, lengths=(100,))
    page_bytes = 8 * 16 * 128 * 2
    pages = (1 << 32) // page_bytes // 2 + step.pages
    cache = A.PagedCache(session, layers=3, pages=pages, kv_heads=8, page_size=16, head_dim=128)
    table = (step.table + (pages - step.pages)).astype(np.uint32)
    for tensor, data in ((cache.keys, step.keys), (cache.values, step.values)):
        part = A.Tensor(session, tensor._buffer, "bf16", data.shape, step_strides(data.shape),
                        (3 * pages - step.pages) * page_bytes // 2)
        set_tensor(part, data)
    batch = A.DraftBatch(upload(session, table, "u32"), upload(session, step.lengths, "u32"), 3)
    got = A.tree_attention(cache, batch, upload(session, step.query, "bf16"), layer=2).storage()
    step.check(got)


def step_strides(shape):
    return [int(np.prod(shape[i + 1:])) for i in range(len(shape))]


def test_captured_calls_follow_new_lengths(session, rng):
    """A captured call is replayed with other lengths, with eager work between."""
    hip = HipRuntime()
    full = Step(rng, B=2, T=4, heads=8, kv=2, dim=128, lengths=(900, 700)).device(session)
    query = upload(session, full.query, "bf16")
    out = session.empty("bf16", query.shape)
    call = lambda: A.tree_attention(full.cache, full.batch, query, out=out)
    call()
    session.synchronize()
    graph = hip.capture(session.stream, call)
    try:
        for lengths in ((900, 700), (33, 0), (899, 650), (1, 2)):
            full.lengths = np.array(lengths, np.uint32)
            set_tensor(full.batch.lengths, full.lengths)
            # the other tokens are NaN for the check's sake only where unseen: all of them are written here
            hip.replay(session.stream, graph)
            replayed = out.storage()
            full.check(replayed)
            call()
            np.testing.assert_array_equal(out.storage(), replayed)
    finally:
        hip.destroy(graph)


@pytest.mark.parametrize("dtype,T", [("bf16", 1), ("bf16", 20), ("f32", 3)])
def test_a_capture_without_scratch(rng, dtype, T):
    """A session's first call, captured: no memory for partial results can be
    had, and every workgroup walks a whole context of several page lists."""
    hip = HipRuntime()
    with A.Session("rocm") as session:
        step = Step(rng, B=2, T=T, heads=8, kv=2, dim=64, lengths=(9000, 4095), dtype=dtype, spread=2.0).device(session)
        query = upload(session, step.query, dtype)
        out = session.empty(dtype, query.shape)
        graph = hip.capture(session.stream, lambda: A.tree_attention(step.cache, step.batch, query, out=out))
        try:
            for _ in range(3):
                hip.replay(session.stream, graph)
                replayed = out.storage()
                step.check(replayed)
                warm = A.tree_attention(step.cache, step.batch, query).storage()  # in pieces
                step.check(warm)
        finally:
            hip.destroy(graph)


def test_calls_from_several_threads(session, rng):
    """Threads share a session's partial results and counters one call at a time."""
    import threading
    steps = [Step(rng, B=1, T=1, heads=8, kv=2, dim=128, lengths=(n,)).device(session) for n in (3000, 900, 5000, 1700)]
    queries = [upload(session, s.query, "bf16") for s in steps]
    results = [[] for _ in steps]

    def work(i):
        for _ in range(20):
            results[i].append(A.tree_attention(steps[i].cache, steps[i].batch, queries[i]))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(steps))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for s, outs in zip(steps, results):
        first = outs[0].storage()
        s.check(first)
        for other in outs[1:]:
            np.testing.assert_array_equal(other.storage(), first)
