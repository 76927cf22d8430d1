"""Outputs that share memory with operands: what is computed in place as it
is elsewhere, and what is refused before anything is enqueued."""
import numpy as np
import pytest

import affon_amd as A
from affon_amd.core import Tensor
from tests.drafts import stored, upload

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
