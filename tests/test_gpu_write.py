"""Tensor.write: new values where calls read them."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import Step, upload
from tests.helpers import HipRuntime

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "u32", "i64"])
def test_values(session, dtype):
    t = session.tensor(np.zeros((4, 6)), dtype)
    values = np.arange(24).reshape(4, 6) * 3
    assert t.write(values) is t
    np.testing.assert_array_equal(t.numpy(), values)
    rows = A.Tensor(session, t._buffer, dtype, (2, 6), (6, 1), 6)  # a contiguous part
    rows.write(np.ones((2, 6)))
    values[1:3] = 1
    np.testing.assert_array_equal(t.numpy(), values)


def test_a_captured_step_with_new_lengths(session, rng):
    hip = HipRuntime()
    step = Step(rng, B=2, T=2, heads=4, kv=2, dim=64, lengths=(40, 90)).device(session)
    query = upload(session, step.query, "bf16")
    out = session.empty("bf16", query.shape)
    A.tree_attention(step.cache, step.batch, query, out=out)
    session.synchronize()
    graph = hip.capture(session.stream, lambda: A.tree_attention(step.cache, step.batch, query, out=out))
    try:
        for lengths in ((40, 90), (0, 33), (39, 1)):
            step.lengths = np.array(lengths, np.uint32)
            step.batch.lengths.write(lengths)
            hip.replay(session.stream, graph)
            step.check(out.storage())
    finally:
        hip.destroy(graph)
