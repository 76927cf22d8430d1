"""Sequences that share a prompt as copies of their own, and are then cut down: from there on they share nothing."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import Step, stored, upload
from tests.test_gpu_weights import evicted

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv,B", [(4, 2, 3), (8, 1, 20)])  # the general kernel's rows, and those of the prefixes' own
@pytest.mark.parametrize("afterwards", [0, 1000])
def test_a_shared_prompt_then_a_budget(session, rng, dtype, heads, kv, B, afterwards):
    prompt, layers = 96, 2
    own = [(7 * b) % 33 for b in range(B)]
    step = Step(rng, B=B, T=1, heads=heads, kv=kv, lengths=[prompt + n for n in own], dtype=dtype, layers=layers, spread=2.0)
    for b in range(1, B):
        for n in range(prompt):
            (to, line), (page, from_line) = step.place(b, n), step.place(0, n)
            for cache in (step.keys, step.values):
                cache[:, to, :, line] = cache[:, page, :, from_line]
    step.device(session)
    shared = upload(session, np.array([prompt], np.uint32), "u32")
    weights = A.token_weights(step.cache, step.batch)
    query = upload(session, step.query, dtype)
    for layer in range(layers):
        step.check(A.shared_attention(step.cache, step.batch, query, shared, layer=layer).storage(), layer=layer)
        A.attention_weights(step.cache, step.batch, query, weights, layer=layer)
    gathered = weights.storage().copy()

    # The drafted tokens are not committed: they go.
    keep, recent = [40 + b for b in range(B)], [8] * B
    A.cache_evict(step.cache, step.batch, weights, upload(session, np.array(keep, np.uint32), "u32"),
                  upload(session, np.array(recent, np.uint32), "u32"), out=weights)
    lengths = np.minimum(step.lengths, np.array(keep, np.uint32))
    keys, values = step.keys.copy(), step.values.copy()
    for layer, b, h in np.ndindex(layers, B, kv):
        kept = evicted(gathered[layer, b, h], int(step.lengths[b]), keep[b], recent[b])
        np.testing.assert_array_equal(weights.storage()[layer, b, h],
                                      np.pad(gathered[layer, b, h, kept], (0, gathered.shape[-1] - len(kept))))
        for to, source in enumerate(kept):
            (p, line), (q, from_line) = step.place(b, to), step.place(b, int(source))
            keys[layer, p, h, line] = step.keys[layer, q, h, from_line]
            values[layer, p, h, line] = step.values[layer, q, h, from_line]
    step.keys, step.values, step.lengths = keys, values, lengths
    step.batch.lengths.write(lengths)

    # The next token, turned by an angle of 0: appended as it is.
    shared.write(np.array([afterwards], np.uint32))
    rotary = upload(session, np.concatenate([np.ones((1, 32)), np.zeros((1, 32))], 1).astype(np.float32), "f32")
    place = upload(session, np.zeros(B, np.uint32), "u32")
    for layer in range(layers):
        key, value = (stored(rng.standard_normal((B, kv * 64)), dtype) for _ in range(2))
        turned = A.cache_append(step.cache, step.batch, query, upload(session, key, dtype), upload(session, value, dtype), place,
                                rotary, layer=layer)
        for b in range(B):
            page, line = step.place(b, int(lengths[b]))
            step.keys[layer, page, :, line], step.values[layer, page, :, line] = key[b].reshape(kv, 64), value[b].reshape(kv, 64)
        step.check(A.shared_attention(step.cache, step.batch, turned, shared, layer=layer).storage(), layer=layer)
