"""The operators over gathered weights, shared prefixes and normed heads as
programs call them: captured and replayed, from several threads, on large
caches, at odd places; and what their Python surface refuses.

Errors of results are bounded as in the tests of each operator."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import Step, mask_words, set_tensor, tree, upload
from tests.helpers import HipRuntime
from tests.test_gpu_shared_attention import share
from tests.test_gpu_tree_attention import step_strides
from tests.test_gpu_weights import check_evict, evicted, gathered
from tests.drafts import U

pytestmark = pytest.mark.gpu


def words(session, values):
    return upload(session, np.array(values, np.uint32), "u32")


class Pipeline:
    """Append with norms and axes, shared attention, gathered weights, an eviction: outputs of a fixed
    state that `reset` brings back."""

    def __init__(self, session, rng, *, T=1, dtype="bf16", lengths=(150, 170, 140), dim=64):
        self.session = session
        self.step = share(Step(rng, B=len(lengths), T=T, heads=4, kv=2, dim=dim, lengths=lengths, dtype=dtype), 1,
                          [128]).device(session)
        # Pages of the prefix are one's own each where tokens move.
        B = len(lengths)
        self.table = np.arange(self.step.table.size, dtype=np.uint32).reshape(B, -1)
        self.moved = A.PagedCache(session, pages=self.table.size, page_size=16, kv_heads=2, head_dim=dim, dtype=dtype)
        self.moved_batch = A.DraftBatch(upload(session, self.table, "u32"), self.step.batch.lengths, T)
        shape = self.moved.keys.shape
        self.start = rng.integers(0, 0x3FFF, shape).astype(np.uint16) if dtype == "bf16" else \
            rng.standard_normal(shape).astype(np.float32)
        R = B * T
        mk = lambda n: upload(session, rng.integers(0x3C00, 0x3FFF, (R, n * dim)).astype(np.uint16), "bf16")
        self.x = mk(4), mk(2), mk(2)
        self.norm = upload(session, np.linspace(0.5, 1.5, dim).astype(np.float32), "f32")
        self.axes = A.rotary_axes((dim // 4, dim // 4))
        self.positions = upload(session, rng.integers(0, 99, (2, R)).astype(np.uint32), "u32")
        self.rotary = A.rotary_table(session, 100, dim)
        self.query = upload(session, self.step.query, dtype)
        self.shared = words(session, [128])
        self.keep, self.recent = words(session, [40] * B), words(session, [9] * B)
        self.gathered = A.token_weights(self.step.cache, self.step.batch)
        self.begin = rng.exponential(size=self.gathered.shape).astype(np.float32)
        self.weights = upload(session, self.begin, "f32")
        self.q = session.empty(dtype, self.query.shape)
        self.attended = session.empty(dtype, self.query.shape)

    def reset(self):
        set_tensor(self.moved.keys, self.start)
        set_tensor(self.moved.values, self.start)
        set_tensor(self.weights, self.begin)
        set_tensor(self.gathered, np.zeros(self.gathered.shape, np.float32))

    def enqueue(self):
        A.cache_append(self.moved, self.moved_batch, *self.x, self.positions, self.rotary, query_norm=self.norm,
                       key_norm=self.norm, axes=self.axes, out=self.q)
        A.shared_attention(self.step.cache, self.step.batch, self.query, self.shared, out=self.attended)
        A.attention_weights(self.step.cache, self.step.batch, self.query, self.gathered)
        A.cache_evict(self.moved, self.moved_batch, self.weights, self.keep, self.recent, out=self.weights)

    def results(self):
        return [t.storage() for t in (self.q, self.attended, self.gathered, self.weights, self.moved.keys, self.moved.values)]

    def eager(self):
        self.reset()
        self.enqueue()
        return self.results()


@pytest.mark.parametrize("T,dtype,dim", [(1, "bf16", 128), (30, "bf16", 64), (5, "f32", 80)])
def test_replays(session, rng, T, dtype, dim):
    """Graphs of two pipelines that share the workspace, replayed in turn with eager calls and other lengths between."""
    hip = HipRuntime()
    both = [Pipeline(session, rng, T=T, dtype=dtype, dim=dim),
            Pipeline(session, rng, T=1 + T // 2, dtype=dtype, dim=dim, lengths=(700, 300, 145))]
    for p in both:
        p.eager()
    graphs = [hip.capture(session.stream, p.enqueue) for p in both]
    try:
        for cut in (0, 3, 100, 0):
            for p, graph in zip(both, graphs):
                set_tensor(p.step.batch.lengths, (p.step.lengths - cut).astype(np.uint32))
                want = p.eager()
                p.reset()
                hip.replay(session.stream, graph)
                for got, expected in zip(p.results(), want):
                    np.testing.assert_array_equal(got, expected)
                if cut == 0:
                    p.step.check(want[1])
        for p in both:
            p.reset()
        for graph in graphs:
            hip.replay(session.stream, graph)
        for p in both:
            replayed = p.results()
            for got, expected in zip(replayed, p.eager()):
                np.testing.assert_array_equal(got, expected)
    finally:
        for graph in graphs:
            hip.destroy(graph)


def test_a_capture_without_workspace(rng):
    """A session's first calls, captured: attention walks each context by itself; the others say what they need."""
    hip = HipRuntime()
    with A.Session("rocm") as session:
        p = Pipeline(session, rng, T=2)
        p.reset()

        def enqueue():
            A.shared_attention(p.step.cache, p.step.batch, p.query, p.shared, out=p.attended)
            with pytest.raises(Exception, match="cache_evict needs a larger workspace.*before the capture"):
                A.cache_evict(p.moved, p.moved_batch, p.weights, p.keep, p.recent, out=p.weights)
            with pytest.raises(Exception, match="attention_weights needs a larger workspace"):
                A.attention_weights(p.step.cache, p.step.batch, p.query, p.gathered)
        graph = hip.capture(session.stream, enqueue)
        try:
            for _ in range(3):
                hip.replay(session.stream, graph)
                p.step.check(p.attended.storage())
                assert not p.gathered.storage().any()
                np.testing.assert_array_equal(p.weights.storage(), p.begin)
                p.step.check(p.eager()[1])
                p.reset()
        finally:
            hip.destroy(graph)


def test_calls_from_several_threads(session, rng):
    import threading
    pipelines = [Pipeline(session, rng, T=t) for t in (1, 3, 20)]
    want = [p.eager() for p in pipelines]
    for p in pipelines:
        p.reset()
    failures = []

    def work(p):
        try:
            p.enqueue()
            for _ in range(10):
                A.shared_attention(p.step.cache, p.step.batch, p.query, p.shared, out=p.attended)
        except Exception as e:  # noqa: BLE001
            failures.append(e)
    threads = [threading.Thread(target=work, args=(p,)) for p in pipelines]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    for p, expected in zip(pipelines, want):
        for got, value in zip(p.results(), expected):
            np.testing.assert_array_equal(got, value)


def check_weights(step, before, got, mask=None):
    total, bound = gathered(step, mask)
    for b in range(step.B):
        length, count = int(step.lengths[b]), int(step.counts[b])
        want = total[b].copy()
        want[:, :length] += before[0, b][:, :length]
        n = length + count if count else 0
        error = np.abs(got[0, b] - want)[:, :n]
        assert (error <= bound[b][:, :n] + U["f32"] * np.abs(want[:, :n])).all()
        np.testing.assert_array_equal(got[0, b][:, n:], before[0, b][:, n:])


@pytest.mark.parametrize("T,dtype", [(1, "bf16"), (12, "bf16"), (60, "f32")])
def test_weights_at_odd_places(session, rng, T, dtype):
    """Weights and queries that begin one value behind a 16-byte boundary."""
    step = Step(rng, B=2, T=T, heads=8, kv=2, dim=72, lengths=(333, 50), dtype=dtype, page=48).device(session)
    shape = (1, 2, 2, step.table.shape[1] * 48)
    size = int(np.prod(shape))
    whole = rng.uniform(0, 2, size + 9).astype(np.float32)
    buffer = upload(session, whole, "f32")
    weights = A.Tensor(session, buffer._buffer, "f32", shape, step_strides(shape), 1)
    wide = np.zeros((2 * T, 8 * 72 + 1), step.query.dtype)
    wide[:, 1:] = step.query
    query = A.slice(upload(session, wide, dtype), [{}, {"start": 1, "stop": 8 * 72 + 1}])
    mask = tree(rng, 2, T)
    A.attention_weights(step.cache, step.batch, query, weights, upload(session, mask_words(mask), "u32"))
    after = buffer.storage()
    check_weights(step, whole[1:1 + size].reshape(shape), after[1:1 + size].reshape(shape), mask)
    np.testing.assert_array_equal(after[1 + size:], whole[1 + size:])
    keep, recent = words(session, [100, 60]), words(session, [30, 0])
    start = after[1:1 + size].reshape(shape)
    A.cache_evict(step.cache, step.batch, weights, keep, recent, out=weights)
    got = buffer.storage()
    want = np.zeros(shape, np.float32)
    for b, h in np.ndindex(2, 2):
        kept = evicted(start[0, b, h], int(step.lengths[b]), (100, 60)[b], (30, 0)[b])
        want[0, b, h, :len(kept)] = start[0, b, h, kept]
    np.testing.assert_array_equal(got[1:1 + size].reshape(shape), want)
    np.testing.assert_array_equal(np.delete(got, slice(1, 1 + size)), np.delete(whole, slice(1, 1 + size)))


def test_a_wide_table(session, rng):
    """A table of more tokens than there is room to keep scores for: few rows' are computed again."""
    step = Step(rng, B=4, T=4, heads=8, kv=2, lengths=(100, 0, 700, 33))
    columns = (1 << 30) // (8 * 16 * 4 * 16) + 1
    table = np.full((4, columns), 0xFFFFFFFF, np.uint32)
    table[:, :step.table.shape[1]] = step.table
    step.table = table
    step.device(session)
    weights = A.token_weights(step.cache, step.batch)
    A.attention_weights(step.cache, step.batch, upload(session, step.query, "bf16"), weights)
    tokens = 50 * 16
    got = A.slice(weights, [{}, {}, {}, {"start": 0, "stop": tokens}]).numpy()
    step.table = table[:, :50]
    check_weights(step, np.zeros((1, 4, 2, tokens), np.float32), got)


@pytest.mark.parametrize("T", [1, 6])
def test_offsets_past_32_bits(session, rng, T):
    """A cache of more than 4 GiB of keys, its tokens at the end: as a small one."""
    step = share(Step(rng, B=3, T=T, heads=8, kv=8, dim=128, lengths=(100, 130, 97)), 1, [96])
    columns, page_bytes = step.table.shape[1], 8 * 16 * 128 * 2
    used = 3 * columns
    assert used >= step.pages
    keys, values = (np.concatenate([data, data[:, :used - step.pages]], 1) for data in (step.keys, step.values))
    query = upload(session, step.query, "bf16")
    norm = upload(session, np.ones(128, np.float32), "f32")
    keep, recent = words(session, [50, 60, 97]), words(session, [10, 10, 10])
    results = []
    for pages in (used, (1 << 32) // page_bytes // 2 + used):
        cache = A.PagedCache(session, pages=pages, kv_heads=8, page_size=16, head_dim=128, layers=3)
        parts = []
        for tensor, data in ((cache.keys, keys), (cache.values, values)):
            parts.append(A.Tensor(session, tensor._buffer, "bf16", data.shape, step_strides(data.shape),
                                  (3 * pages - used) * page_bytes // 2))
            set_tensor(parts[-1], data)
        batch = A.DraftBatch(upload(session, (step.table + (pages - used)).astype(np.uint32), "u32"),
                             upload(session, step.lengths, "u32"), T)
        attended = A.shared_attention(cache, batch, query, words(session, [96]), layer=2)
        weights = A.token_weights(cache, batch)
        A.attention_weights(cache, batch, query, weights, layer=2)
        gathered_by = weights.storage()
        q = A.cache_append(cache, batch, query, query, query, None, A.rotary_table(session, 200, 128), layer=2,
                           query_norm=norm, key_norm=norm)
        results.append([attended.storage(), gathered_by, q.storage(), *(t.storage() for t in parts)])
        # An eviction takes pages of each sequence's own.
        own = A.DraftBatch(upload(session, (np.arange(used).reshape(3, columns) + pages - used).astype(np.uint32), "u32"),
                           batch.lengths, T)
        A.cache_evict(cache, own, weights, keep, recent, out=weights)
        results[-1] += [weights.storage(), *(t.storage() for t in parts)]
    step.check(results[0][0])
    for small, large in zip(*results):
        np.testing.assert_array_equal(small, large)


def test_evictions_of_every_page_size(session, rng):
    for page in (16, 32, 80, 112, 1024, 4096, 8192):
        check_evict(session, rng, lengths=(page + 40, 5), keep=(page // 2 + 1, 5), recent=(page // 4, 1), page=page, dim=8,
                    layers=1)


def test_refusals(session):
    cache = A.PagedCache(session, pages=4, page_size=16, kv_heads=2, head_dim=8, layers=2)
    batch = A.DraftBatch(session.empty("u32", (2, 2)), session.empty("u32", (2,)), 3)
    query, kv = session.empty("bf16", (6, 32)), session.empty("bf16", (6, 16))
    rotary, two = session.empty("f32", (10, 8)), session.empty("u32", (2,))
    weights = A.token_weights(cache, batch)
    assert weights.shape == (2, 2, 2, 32)
    f32 = lambda *shape: session.empty("f32", shape)
    for options, message in (({"query_norm": f32(9)}, "query_norm must be"), ({"key_norm": f32(32)}, "key_norm must be"),
                             ({"query_norm": session.empty("u32", (8,))}, "query_norm must be"),
                             ({"axes": (0, 0, 1, 1)}, "RotaryAxes"), ({"axes": A.RotaryAxes([0, 1])}, "rotary_dim / 2 pairs"),
                             ({"query_norm": f32(8), "epsilon": 0.0}, "epsilon"),
                             ({"query_norm": f32(8), "epsilon": float("nan")}, "epsilon")):
        with pytest.raises(Exception, match=message):
            A.cache_append(cache, batch, query, kv, kv, None, rotary, **options)
    with pytest.raises(TypeError, match="positions must be"):
        A.cache_append(cache, batch, query, kv, kv, session.empty("u32", (6,)), rotary, axes=A.rotary_axes((2, 2)))
    with pytest.raises(Exception, match="overlaps"):
        A.cache_append(cache, batch, query, kv, kv, None, rotary, query_norm=f32(8), out=A.Tensor(
            session, cache.keys._buffer, "bf16", (6, 32), [32, 1], 0))
    for shared in (session.empty("u32", (3,)), session.empty("u32", (0,)), session.empty("u32", (1, 1)),
                   session.empty("f32", (1,)), None):
        with pytest.raises(TypeError, match="shared"):
            A.shared_attention(cache, batch, query, shared)
    one = session.empty("u32", (1,))
    for args, options, message in (((session.empty("f32", (6, 32)), one), {}, "query"), ((query, one), {"layer": 2}, "layer"),
                                   ((query, one, session.empty("u32", (5, 1))), {}, "mask"),
                                   ((query, one), {"scale": float("inf")}, "scale"),
                                   ((query, one), {"out": session.empty("bf16", (6, 16))}, "output")):
        with pytest.raises(Exception, match=message):
            A.shared_attention(cache, batch, *args, **options)
    for args, options, message in (((query, f32(2, 2, 2, 31)), {}, "weights must be"), ((query, None), {}, "weights must be"),
                                   ((session.empty("bf16", (6, 24)), weights), {}, "multiple of kv_heads"),
                                   ((query, weights, session.empty("f32", (6, 1))), {}, "mask"),
                                   ((query, weights), {"scale": float("nan")}, "scale"),
                                   ((query, A.Tensor(session, cache.values._buffer, "f32", weights.shape,
                                                     step_strides(weights.shape), 0)), {}, "overlap")):
        with pytest.raises(Exception, match=message):
            A.attention_weights(cache, batch, *args, **options)
    twice = f32(2 * 256 + 8)
    at = lambda n: A.Tensor(session, twice._buffer, "f32", weights.shape, step_strides(weights.shape), n)
    for args, options, message in (((f32(2, 2, 2, 16), two, two), {}, "weights must be"), ((weights, one, two), {}, "keep"),
                                   ((weights, two, f32(2)), {}, "recent"), ((at(0), two, two), {"out": at(8)}, "overlaps"),
                                   ((weights, two, two), {"out": f32(2, 2, 2, 16)}, "output")):
        with pytest.raises(Exception, match=message):
            A.cache_evict(cache, batch, *args, **options)
    path = session.empty("u32", (2, 2))
    with pytest.raises(TypeError, match="weights must be"):
        A.cache_commit(cache, batch, path, two, weights=f32(2, 2, 2, 16))
    with A.Session("rocm") as other:
        with pytest.raises(TypeError, match="same Session"):
            A.attention_weights(cache, batch, query, other.empty("f32", weights.shape))
        with pytest.raises(TypeError, match="same Session"):
            A.cache_append(cache, batch, query, kv, kv, None, rotary, query_norm=other.empty("f32", (8,)))
        with pytest.raises(TypeError, match="same Session"):
            A.cache_evict(cache, batch, weights, two, other.empty("u32", (2,)))


@pytest.mark.parametrize("B,groups,dtype", [(17, 1, "bf16"), (34, 2, "f32"), (3, 1, "bf16")])
def test_tables_of_almost_2_to_the_31_tokens(session, rng, B, groups, dtype):
    """Prefixes of as many tokens, of which the first page's alone lie anywhere: keys of 0, so
    that the mean of their values is the result. The values are small integers, whose sums are exact
    in f32 in any order; the quotient is rounded, and to bf16 again."""
    page, columns = 65536, 32767
    cache = A.PagedCache(session, pages=2, page_size=page, kv_heads=1, head_dim=64, dtype=dtype)
    values = rng.integers(0, 5, (1, 2, 1, page, 64)).astype(np.float32)
    values[..., :32] = 4
    half = dtype == "bf16"
    set_tensor(cache.keys, np.zeros(values.shape, np.uint16 if half else np.float32))
    set_tensor(cache.values, (values.view(np.uint32) >> 16).astype(np.uint16) if half else values)
    table = np.full((B, columns), 0xFFFFFFFF, np.uint32)
    table[:, 0] = 1
    tokens = page * columns
    lengths = np.full(B, tokens - 5000, np.uint32)
    shared = np.full(groups, tokens - 70000, np.uint32)
    shared[1:] = 0
    batch = A.DraftBatch(upload(session, table, "u32"), upload(session, lengths, "u32"), 1)
    query = session.tensor(rng.standard_normal((B, 64)), dtype)
    got = A.shared_attention(cache, batch, query, upload(session, shared, "u32")).numpy()
    want = np.broadcast_to(values[0, 1, 0].mean(0, dtype=np.float64), got.shape)
    np.testing.assert_allclose(got, want, rtol=2.0 ** -8 + 2.0 ** -20 if half else 2.0 ** -20)
