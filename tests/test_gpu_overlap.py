"""Outputs that share memory with operands: what is computed in place as it
is elsewhere, and what is refused before anything is enqueued."""
import numpy as np
import pytest

import affon_amd as A
from affon_amd.core import Tensor
from tests.drafts import Step, stored, upload

pytestmark = pytest.mark.gpu


def view(t, shape, strides, offset=0, dtype=None):
    return Tensor(t.session, t._buffer, dtype or t.dtype, shape, strides, offset)


@pytest.mark.parametrize("N", [40, 20000])
@pytest.mark.parametrize("post", [False, True])
def test_norms_in_place_of_each_operand(session, rng, N, post):
    make = lambda: [upload(session, a, "f32") for a in arrays]
    arrays = [stored(rng.standard_normal((5, N)), "f32") for _ in range(3)]
    x, u, g = make()
    want = [t.numpy() for t in A.residual_norm(x, u, gate=g, post_norm=post)]
    for first in range(4):
        for second in range(4):
            operands = make()
            spare = session.empty("f32", (5, N)), session.empty("f32", (5, N))
            out = tuple(operands[i] if i < 3 else s for i, s in zip((first, second), spare))
            if first == second < 3:
                with pytest.raises(TypeError, match="outputs overlap"):
                    A.residual_norm(operands[0], operands[1], gate=operands[2], post_norm=post, out=out)
                for t, a in zip(operands, arrays):
                    np.testing.assert_array_equal(t.numpy(), a)
                continue
            got = A.residual_norm(operands[0], operands[1], gate=operands[2], post_norm=post, out=out)
            for t, w in zip(got, want):
                np.testing.assert_array_equal(t.numpy(), w)


def test_norms_of_columns_of_one_tensor(session, rng):
    """Rows that lie between each other and share nothing."""
    N, wide = 24, stored(rng.standard_normal((6, 4 * 24)), "f32")
    whole = upload(session, wide, "f32")
    x, u, y, n = (view(whole, (6, N), (4 * N, 1), i * N) for i in range(4))
    want = [t.numpy() for t in A.residual_norm(upload(session, wide[:, :N], "f32"), upload(session, wide[:, N:2 * N], "f32"))]
    A.residual_norm(x, u, out=(y, n))
    np.testing.assert_array_equal(whole.numpy(), np.concatenate([wide[:, :2 * N], *want], 1))


def test_norms_whose_outputs_overlap(session, rng):
    data = stored(rng.standard_normal((16, 64)), "f32")
    whole = upload(session, data, "f32")
    x = view(whole, (4, 32), (64, 1))
    u = upload(session, data[:4, :32], "f32")
    spare = lambda: session.empty("f32", (4, 32))
    for out, message in (((x, x), "outputs overlap"),
                         ((spare(), view(whole, (4, 32), (32, 1))), "overlaps an operand"),  # another stride
                         ((view(whole, (4, 32), (64, 1), 1), spare()), "overlaps an operand"),  # a value further
                         ((view(whole, (4, 32), (64, 1), 64), spare()), "overlaps an operand"),  # a row further
                         ((spare(), view(whole, (4, 32), (64, 1), 0, "bf16")), "overlaps an operand")):
        for args in ((x, u), (x,)):
            with pytest.raises(TypeError, match=message):
                A.residual_norm(*args, out=out)
    weight = view(whole, (32,), (1,), 64 * 8)
    for options in ({"weight": weight}, {"gate": weight}, {"post_norm": True, "post_weight": weight}):
        with pytest.raises(TypeError, match="overlaps an operand"):
            A.residual_norm(x, u, out=(spare(), view(whole, (4, 32), (64, 1), 64 * 6)), **options)
    np.testing.assert_array_equal(whole.numpy(), data)


def test_norms_without_an_update(session, rng):
    """A first output at the stream's address with another stride is not the
    stream, and rows at stride 0 are no reason to refuse a stream that is kept."""
    data = stored(rng.standard_normal((8, 64)), "f32")
    whole = upload(session, data, "f32")
    with pytest.raises(TypeError, match="overlaps an operand"):
        A.residual_norm(view(whole, (4, 32), (64, 1)), out=(view(whole, (4, 32), (32, 1)), session.empty("f32", (4, 32))))
    np.testing.assert_array_equal(whole.numpy(), data)
    row = view(whole, (4, 64), (0, 1))
    same, n = A.residual_norm(row)
    assert same is row
    one = A.residual_norm(view(whole, (1, 64), (64, 1)))[1].numpy()
    np.testing.assert_array_equal(n.numpy(), np.repeat(one, 4, axis=0))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,lengths", [(1, (700, 3)), (40, (50, 0)), (70, (2500, 900))])
def test_attention_and_append_in_place_of_the_query(session, rng, dtype, T, lengths):
    step = Step(rng, B=2, T=T, heads=8, kv=2, dim=64, lengths=lengths, dtype=dtype).device(session)
    query = lambda: upload(session, step.query, dtype)
    want = A.tree_attention(step.cache, step.batch, query()).storage()
    step.check(want)
    q = query()
    assert A.tree_attention(step.cache, step.batch, q, out=q) is q
    np.testing.assert_array_equal(q.storage(), want)
    for interleaved in (False, True):
        args = (query(), query(), None, A.rotary_table(session, 4000, 64))
        kv = [upload(session, step.query[:, i * 128:(i + 1) * 128], dtype) for i in range(2)]
        want = A.cache_append(step.cache, step.batch, query(), *kv, *args[2:], interleaved=interleaved).storage()
        q = query()
        A.cache_append(step.cache, step.batch, q, *kv, *args[2:], interleaved=interleaved, out=q)
        np.testing.assert_array_equal(q.storage(), want)


def test_outputs_that_overlap_operands(session, rng):
    step = Step(rng, B=2, T=3, heads=4, kv=2, dim=64, lengths=(20, 7)).device(session)
    wide = session.empty("bf16", (20, 512))
    columns = view(wide, (6, 256), (512, 1))
    refused = lambda: pytest.raises(Exception, match="overlaps an operand")
    with refused():  # the same first row, another stride
        A.tree_attention(step.cache, step.batch, columns, out=view(wide, (6, 256), (256, 1)))
    query = view(wide, (6, 256), (256, 1))
    with refused():  # a row further
        A.tree_attention(step.cache, step.batch, query, out=view(wide, (6, 256), (256, 1), 256))
    whole = step.cache.keys
    flat = view(whole, (6, 256), (256, 1), 64)
    keys = whole.storage()
    kv = [upload(session, step.query[:, :128], "bf16") for _ in range(2)]
    rotary = A.rotary_table(session, 64, 64)
    for out in (flat, view(step.cache.values, (6, 256), (256, 1))):
        with refused():
            A.tree_attention(step.cache, step.batch, query, out=out)
        with refused():
            A.cache_append(step.cache, step.batch, query, *kv, None, rotary, out=out)
    with refused():  # a value that is part of the output
        A.cache_append(step.cache, step.batch, upload(session, step.query, "bf16"), kv[0], view(wide, (6, 128), (512, 1), 128),
                       None, rotary, out=query)
    with refused():  # f32 queries where bf16 ones go
        f32 = session.empty("f32", (6, 256))
        A.cache_append(step.cache, step.batch, f32, *(view(session.empty("f32", (6, 128)), (6, 128), (128, 1)) for _ in "kv"),
                       None, rotary, out=view(f32, (6, 256), (256, 1), 0, "bf16"))
    np.testing.assert_array_equal(whole.storage(), keys)
    # Columns beside the query's are no part of it.
    data = np.zeros((6, 512), np.uint16)
    data[:, :256] = step.query
    part = upload(session, data, "bf16")
    A.tree_attention(step.cache, step.batch, view(part, (6, 256), (512, 1)), out=view(wide, (6, 256), (256, 1)))
