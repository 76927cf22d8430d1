"""Gathered weights of tokens that have gathered none."""
import tracemalloc

import numpy as np
import pytest

import affon_amd as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layers,B,kv,page,columns", [(1, 1, 1, 16, 1), (3, 5, 2, 48, 7), (2, 1, 3, 1008, 37)])
def test_zeros(session, layers, B, kv, page, columns):
    cache = A.PagedCache(session, pages=2, page_size=page, kv_heads=kv, head_dim=8, layers=layers)
    batch = A.DraftBatch(session.empty("u32", (B, columns)), session.empty("u32", (B,)), 1)
    shape = (layers, B, kv, columns * page)
    for _ in range(3):  # where other values were before
        session.tensor(np.ones(shape), "f32")
    weights = A.token_weights(cache, batch)
    assert weights.shape == shape and weights.dtype == "f32"
    assert not weights.storage().view(np.uint32).any()


def test_made_on_the_device(session):
    """128 MB of weights take no host memory."""
    cache = A.PagedCache(session, pages=1, page_size=16, kv_heads=8, head_dim=8, layers=32)
    batch = A.DraftBatch(session.empty("u32", (2, 4096)), session.empty("u32", (2,)), 1)
    tracemalloc.start()
    try:
        weights = A.token_weights(cache, batch)
        session.synchronize()
        peak = tracemalloc.get_traced_memory()[1]
    finally:
        tracemalloc.stop()
    assert peak < 1 << 20
    assert not weights.storage().view(np.uint32).any()
