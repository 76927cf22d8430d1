"""What the Python surface of the drafted-token ops and residual_norm refuses."""
import numpy as np
import pytest

import affon_amd as A

pytestmark = pytest.mark.gpu


def test_caches_and_batches(session):
    for changes, message in (({"pages": 0}, "pages"), ({"page_size": 20}, "multiple of 16"),
                             ({"head_dim": 12}, "multiple of 8"), ({"head_dim": 512}, "at most 256"),
                             ({"dtype": "u32"}, "f32 or bf16"), ({"layers": True}, "layers")):
        with pytest.raises(TypeError, match=message):
            A.PagedCache(session, **({"pages": 4, "page_size": 16, "kv_heads": 1, "head_dim": 8} | changes))
    table, lengths = session.empty("u32", (2, 3)), session.empty("u32", (2,))
    with pytest.raises(TypeError, match="page_table"):
        A.DraftBatch(session.empty("f32", (2, 3)), lengths, 1)
    with pytest.raises(TypeError, match="lengths"):
        A.DraftBatch(table, session.empty("u32", (3,)), 1)
    with pytest.raises(TypeError, match="counts"):
        A.DraftBatch(table, lengths, 1, counts=session.empty("i64", (2,)))
    with pytest.raises(TypeError, match="rows"):
        A.DraftBatch(table, lengths, 0)


def test_calls(session):
    cache = A.PagedCache(session, pages=4, page_size=16, kv_heads=2, head_dim=8)
    batch = A.DraftBatch(session.empty("u32", (2, 2)), session.empty("u32", (2,)), 3)
    query, kv = session.empty("bf16", (6, 32)), session.empty("bf16", (6, 16))
    rotary = session.empty("f32", (10, 8))
    for args, options, message in (
            ((session.empty("bf16", (6, 24)), kv, kv, None, rotary), {}, "multiple of kv_heads"),
            ((session.empty("bf16", (5, 32)), kv, kv, None, rotary), {}, "query"),
            ((query, session.empty("f32", (6, 16)), kv, None, rotary), {}, "key"),
            ((query, kv, session.empty("bf16", (6, 8)), None, rotary), {}, "value"),
            ((query, kv, kv, session.empty("u32", (5,)), rotary), {}, "positions"),
            ((query, kv, kv, None, session.empty("f32", (10, 10))), {}, "rotary"),
            ((query, kv, kv, None, rotary), {"layer": 1}, "layer"),
            ((query, kv, kv, None, rotary), {"out": session.empty("f32", (6, 32))}, "output"),
            ((A.transpose(session.empty("bf16", (32, 6)), (1, 0)), kv, kv, None, rotary), {}, "consecutive")):
        with pytest.raises(TypeError, match=message):
            A.cache_append(cache, batch, *args, **options)
    for args, options, message in (
            ((session.empty("f32", (6, 32)),), {}, "query"), ((query, session.empty("u32", (5, 1))), {}, "mask"),
            ((query, session.empty("f32", (6, 1))), {}, "mask"), ((query,), {"layer": -1}, "layer"),
            ((query,), {"out": session.empty("bf16", (6, 16))}, "output")):
        with pytest.raises(TypeError, match=message):
            A.tree_attention(cache, batch, *args, **options)
    with pytest.raises(Exception, match="scale"):
        A.tree_attention(cache, batch, query, scale=float("nan"))
    with pytest.raises(TypeError, match="bit for every row"):
        wide = A.DraftBatch(batch.page_table, batch.lengths, 40)
        A.tree_attention(cache, wide, session.empty("bf16", (80, 32)), session.empty("u32", (80, 1)))
    accepted = session.empty("u32", (2,))
    for path, message in ((session.empty("u32", (2, 4)), "longer"), (session.empty("u32", (3, 2)), "path")):
        with pytest.raises(TypeError, match=message):
            A.cache_commit(cache, batch, path, accepted)
    with pytest.raises(TypeError, match="accepted"):
        A.cache_commit(cache, batch, session.empty("u32", (2, 2)), session.empty("u32", (3,)))
    with A.Session("rocm") as other:
        with pytest.raises(TypeError, match="same Session"):
            A.tree_attention(cache, batch, other.empty("bf16", (6, 32)))
    with pytest.raises(TypeError, match="rotary_dim"):
        A.rotary_table(session, 4, 7)
    gone = A.PagedCache(session, pages=4, page_size=16, kv_heads=2, head_dim=8)
    gone.keys.dispose()
    with pytest.raises(RuntimeError, match="disposed"):
        A.tree_attention(gone, batch, query)


def test_norms(session):
    x = session.tensor(np.ones((3, 8)), "f32")
    for args, options, message in (
            ((session.empty("f32", (8,)),), {}, "rank-two"), ((session.empty("u32", (3, 8)),), {}, "stream"),
            ((x, session.empty("f32", (3, 7))), {}, "update"), ((x, x), {"gate": session.empty("f32", (3,))}, "gate"),
            ((x,), {"gate": x}, "no gate"), ((x,), {"post_norm": True}, "no post_norm"),
            ((x, x), {"post_weight": session.empty("f32", (8,))}, "needs post_norm"),
            ((x, x), {"weight": session.empty("f32", (7,))}, "weight"), ((x, x), {"epsilon": 0.0}, "epsilon"),
            ((x, x), {"scale": float("inf")}, "scale"), ((x, x), {"dtype": "u32"}, "f32 or bf16"),
            ((x, x), {"out": (session.empty("bf16", (3, 8)), x)}, "outputs"),
            ((x, x), {"weight": session.empty("f32", (8,)), "post_norm": True,
                      "post_weight": session.empty("bf16", (8,))}, "one type"),
            ((x, A.transpose(session.empty("f32", (8, 3)), (1, 0))), {}, "consecutive")):
        with pytest.raises(TypeError, match=message):
            A.residual_norm(*args, **options)
