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
