"""Captured attention calls whose pieces are few: replays give what eager
calls give, bit for bit, and leave nothing behind for them."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import Step, set_tensor, upload
from tests.helpers import HipRuntime

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,B,heads,kv,dim,lengths", [
    ("bf16", 1, 32, 8, 128, (777,)), ("bf16", 1, 8, 8, 64, (5000,)), ("f32", 2, 4, 2, 64, (900, 31)),
    ("bf16", 3, 8, 2, 128, (700, 1500, 2))])
def test_replays_beside_eager_calls(session, rng, dtype, B, heads, kv, dim, lengths):
    hip = HipRuntime()
    step = Step(rng, B=B, heads=heads, kv=kv, dim=dim, lengths=lengths, dtype=dtype).device(session)
    query = upload(session, step.query, dtype)
    out, eager = session.empty(dtype, query.shape), session.empty(dtype, query.shape)
    call = lambda to: A.tree_attention(step.cache, step.batch, query, out=to)
    call(eager)
    session.synchronize()
    graph = hip.capture(session.stream, lambda: call(out))
    try:
        for cut in (0, 0, 1, 40, 0):
            step.lengths = np.array([max(0, n - cut) for n in lengths], np.uint32)
            set_tensor(step.batch.lengths, step.lengths)
            hip.replay(session.stream, graph)
            call(eager)
            replayed = out.storage()
            step.check(replayed)
            np.testing.assert_array_equal(eager.storage(), replayed)
            call(eager)
            np.testing.assert_array_equal(eager.storage(), replayed)
    finally:
        hip.destroy(graph)
