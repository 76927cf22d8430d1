"""Drafted trees whose weights are gathered, committed with their tokens and then cut down: the readme's loop."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import Step, mask_words, tree, upload
from tests.test_gpu_weights import evicted, gathered

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T", [5, 24])
def test_commit_then_evict(session, rng, dtype, T):
    B, kv, layers, lengths = 3, 2, 2, [70, 33, 0]
    step = Step(rng, B=B, T=T, heads=4, kv=kv, lengths=lengths, counts=[T, T - 2, T], dtype=dtype, layers=layers,
                spread=2.0).device(session)
    mask = tree(rng, B, T)
    words = upload(session, mask_words(mask), "u32")
    weights = A.token_weights(step.cache, step.batch)
    query = upload(session, step.query, dtype)
    for layer in range(layers):
        A.attention_weights(step.cache, step.batch, query, weights, words, layer=layer)
        total, bound = gathered(step, mask, layer=layer)
        got = weights.storage()[layer]
        assert (np.abs(got - total) <= bound + 2.0 ** -24 * total).all()
    want = weights.storage().copy()

    # The deepest drafted token's ancestors are accepted.
    path, accepted = np.zeros((B, T), np.uint32), np.zeros(B, np.uint32)
    for b in range(B):
        own = mask[b * T:b * T + int(step.counts[b])]
        walk = np.nonzero(own[own.sum(1).argmax()])[0]
        path[b, :len(walk)], accepted[b] = walk, len(walk)
    path_device = upload(session, path, "u32")
    A.cache_commit(step.cache, step.batch, path_device, upload(session, accepted, "u32"), weights=weights)
    source = [np.concatenate([np.arange(n), n + path[b, :accepted[b]]]).astype(int) for b, n in enumerate(lengths)]
    committed = np.zeros_like(want)
    for b in range(B):
        committed[:, b, :, :len(source[b])] = want[:, b][..., source[b]]
    np.testing.assert_array_equal(weights.storage(), committed)

    now = np.array(lengths) + accepted
    step.batch.lengths.write(now.astype(np.uint32))
    keep, recent = [40, 36, 2], [8, 40, 1]
    A.cache_evict(step.cache, step.batch, weights, upload(session, np.array(keep, np.uint32), "u32"),
                  upload(session, np.array(recent, np.uint32), "u32"), out=weights)
    left, keys, values = weights.storage(), step.cache.keys.storage(), step.cache.values.storage()
    for layer, b, h in np.ndindex(layers, B, kv):
        kept = evicted(committed[layer, b, h], int(now[b]), keep[b], recent[b])
        np.testing.assert_array_equal(left[layer, b, h], np.pad(committed[layer, b, h, kept], (0, left.shape[-1] - len(kept))))
        for to, n in enumerate(source[b][kept]):
            (p, line), (q, from_line) = step.place(b, to), step.place(b, int(n))
            np.testing.assert_array_equal(keys[layer, p, h, line], step.keys[layer, q, h, from_line])
            np.testing.assert_array_equal(values[layer, p, h, line], step.values[layer, q, h, from_line])
