"""Gathered weights and shared prefixes of more sequences, or groups, than a wave has lanes, and of long
pieces of prompts; evictions at every step."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import Step, tree, upload
from tests.test_gpu_shared_attention import run, share
from tests.test_gpu_weights import check, evicted

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,T,heads,kv", [(65, 1, 4, 2), (130, 3, 4, 1), (200, 1, 2, 2), (70, 20, 4, 2), (129, 9, 8, 1)])
@pytest.mark.parametrize("in_use", ["most", "late", "one"])
def test_weights(session, rng, dtype, B, T, heads, kv, in_use):
    """The first sequences with rows in use are the first, those past a wave's lanes, or the last alone."""
    lengths = rng.integers(0, 300, B)
    lengths[rng.integers(0, B, 5)] = 0
    counts = rng.integers(0, T + 1, B)
    counts[-1] = T
    counts[:{"most": 0, "late": 64, "one": B - 1}[in_use]] = 0
    check(session, rng, Step(rng, B=B, T=T, heads=heads, kv=kv, lengths=lengths, counts=counts, dtype=dtype, spread=2.0))


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("bf16", 72), ("f32", 64)])
@pytest.mark.parametrize("groups,per,T,heads,kv", [(70, 1, 1, 4, 2), (65, 3, 2, 4, 1), (130, 5, 1, 4, 1), (66, 9, 2, 8, 1)])
def test_shared(session, rng, dtype, dim, groups, per, T, heads, kv):
    """Prefixes of many groups, from none to some hundred tokens; some long, some sequences without them."""
    shared = rng.integers(0, 200, groups)
    shared[rng.integers(0, groups, 4)] = 1500
    shared[rng.integers(0, groups, 4)] = 0
    B = groups * per
    lengths = np.repeat(shared, per) + rng.integers(0, 40, B)
    short = rng.integers(0, B, B // 8)
    short = short[short % per != 0]
    lengths[short] //= 3
    step = share(Step(rng, B=B, T=T, heads=heads, kv=kv, dim=dim, lengths=lengths, counts=rng.integers(0, T + 1, B), dtype=dtype,
                      spread=2.0), groups, shared).device(session)
    used = (np.arange(T) < step.counts[:, None]).reshape(-1)
    got = run(session, step, shared)
    assert not got[~used].any()
    step.check(got, rows=used)


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("bf16", 128), ("bf16", 96), ("f32", 80)])
@pytest.mark.parametrize("masked", [False, True])
def test_long_pieces_after_a_prefix(session, rng, dtype, dim, masked):
    """Each sequence's own prompt after the system's."""
    step = share(Step(rng, B=2, T=300, heads=4, kv=2, dim=dim, lengths=[500, 517], counts=[300, 261], dtype=dtype, spread=2.0),
                 1, [500]).device(session)
    mask = tree(rng, 2, 300, 0.1) if masked else None
    step.check(run(session, step, [500], mask), mask)


@pytest.mark.parametrize("page,length", [(16, 150), (48, 4200)])
def test_an_eviction_at_every_step(session, rng, page, length):
    """A budget that is held token by token: the one of the least weight goes, lines and weights follow."""
    B, kv, steps = 2, 2, 12
    step = Step(rng, B=B, T=1, kv=kv, heads=kv, page=page, lengths=[length, length - 7]).device(session)
    shape = (1, B, kv, step.table.shape[1] * page)
    held = rng.exponential(size=shape).astype(np.float32)
    for b in range(B):
        held[:, b, :, int(step.lengths[b]):] = 0
    weights = upload(session, held, "f32")
    lengths = step.lengths.astype(int)
    order = [[np.arange(n) for _ in range(kv)] for n in lengths]  # the tokens that are left
    for _ in range(steps):
        keep = upload(session, (lengths - 1).astype(np.uint32), "u32")
        before = weights.storage().copy()
        A.cache_evict(step.cache, step.batch, weights, keep, upload(session, np.full(B, 3, np.uint32), "u32"), out=weights)
        for b, h in np.ndindex(B, kv):
            kept = evicted(before[0, b, h], int(lengths[b]), int(lengths[b]) - 1, 3)
            order[b][h] = order[b][h][kept]
        lengths = lengths - 1
        step.batch.lengths.write(lengths.astype(np.uint32))
    got, keys, values = weights.storage(), step.cache.keys.storage(), step.cache.values.storage()
    for b, h in np.ndindex(B, kv):
        n = int(lengths[b])
        np.testing.assert_array_equal(got[0, b, h], np.pad(held[0, b, h, order[b][h]], (0, shape[-1] - n)))
        for to, source in enumerate(order[b][h]):
            (p, line), (q, from_line) = step.place(b, to), step.place(b, int(source))
            np.testing.assert_array_equal(keys[0, p, h, line], step.keys[0, q, h, from_line])
            np.testing.assert_array_equal(values[0, p, h, line], step.values[0, q, h, from_line])
