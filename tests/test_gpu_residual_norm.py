"""residual_norm on the GPU against the formula in 64 bits. The sums of a row
are added in parts of at most 64 values, so that a norm's relative error is
under 48 f32 roundings (half of the sum's 64, and those of the mean, the root
and the products); a result is rounded once more to its type."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import U, stored, upload, widened

pytestmark = pytest.mark.gpu

NORM = 48 * U["f32"]


def check(session, rng, M, N, *, stream="f32", update="f32", out="bf16", weight="bf16", gate=None, gate_dtype="f32",
          post=False, scale=1.0, epsilon=1e-5, in_place=False, pad=0):
    x, u = stored(rng.standard_normal((M, N + pad)) * 2, stream), stored(rng.standard_normal((M, N + pad)), update)
    w, pw = (stored(1 + 0.2 * rng.standard_normal(N), weight) for _ in range(2))
    g = None if gate is None else stored(rng.standard_normal((N,) if gate == "columns" else (M, N + pad)), gate_dtype)
    cut = lambda t: A.slice(t, [{}, {"start": pad}]) if len(t.shape) == 2 else t
    xt, ut = cut(upload(session, x, stream)), cut(upload(session, u, update))
    options = {"weight": upload(session, w, weight), "scale": scale, "epsilon": epsilon, "dtype": out}
    if post:
        options |= {"post_norm": True, "post_weight": upload(session, pw, weight)}
    if g is not None:
        options["gate"] = cut(upload(session, g, gate_dtype))
    if in_place:
        options["out"] = (xt, session.empty(out, (M, N)))
    got_x, got_n = A.residual_norm(xt, ut, **options)
    x, u = widened(x)[:, pad:], widened(u)[:, pad:]
    u0 = u
    if post:
        u0 = u0 / np.sqrt((u0 ** 2).mean(1, keepdims=True) + epsilon) * widened(pw)
    if g is not None:
        u0 = u0 * (widened(g) if gate == "columns" else widened(g)[:, pad:])
    y = x + scale * u0
    n = y / np.sqrt((y ** 2).mean(1, keepdims=True) + epsilon)
    slack = (NORM + 4 * U["f32"]) * np.abs(scale * u0) + 2 * U["f32"] * np.abs(y)  # of stream', before it is rounded
    assert (np.abs(widened(got_x.storage()) - y) <= slack + U[stream] * (np.abs(y) + slack)).all()
    per = np.abs(widened(w)) / np.sqrt((y ** 2).mean(1, keepdims=True) + epsilon)
    # An error of the values, and that of their norm (at most their root mean square error over the norm).
    shift = np.sqrt((slack ** 2).mean(1, keepdims=True) / ((y ** 2).mean(1, keepdims=True) + epsilon))
    n = n * widened(w)
    bound = slack * per + (NORM + 2 * shift) * np.abs(n)
    assert (np.abs(widened(got_n.storage()) - n) <= bound + U[out] * (np.abs(n) + bound)).all()


@pytest.mark.parametrize("N", [1, 7, 8, 65, 512, 513, 1000, 2048, 4096, 4100, 8192, 8200, 16384, 16385, 40000])
def test_widths(session, rng, N):
    check(session, rng, 3, N)
    check(session, rng, 2, N, post=True, gate="rows", scale=0.5, stream="bf16", update="bf16", out="f32", weight="f32")


@pytest.mark.parametrize("stream", ["f32", "bf16"])
@pytest.mark.parametrize("update", ["f32", "bf16"])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_types(session, rng, stream, update, out):
    for gate, post in ((None, False), ("columns", True), ("rows", False)):
        for weight in ("f32", "bf16"):
            check(session, rng, 5, 300, stream=stream, update=update, out=out, weight=weight, gate=gate, post=post,
                  gate_dtype="bf16", scale=0.22)


@pytest.mark.parametrize("N", [96, 4096, 20000])
def test_in_place_and_strided(session, rng, N):
    for pad in (0, 1, 5):
        check(session, rng, 4, N, in_place=True, post=True, pad=pad, gate="rows")
        check(session, rng, 4, N, in_place=True, pad=pad, stream="bf16", gate="rows", gate_dtype="bf16")


def test_many_rows(session, rng):
    check(session, rng, 3000, 40)
    check(session, rng, 1500, 1024, stream="bf16")


def test_weights_and_update_left_out(session, rng):
    """No update: a norm with a weight; no weights: the framework's rms_norm."""
    x = upload(session, stored(rng.standard_normal((3, 200)), "f32"), "f32")
    w = upload(session, stored(rng.standard_normal(200), "f32"), "f32")
    same, n = A.residual_norm(x, weight=w)
    assert same is x
    plain = A.rms_norm(x, -1).numpy().astype(np.float64)
    np.testing.assert_allclose(n.numpy(), plain * w.numpy(), rtol=3 * NORM)
    copy, n = A.residual_norm(x, out=(session.empty("f32", (3, 200)), session.empty("f32", (3, 200))))
    np.testing.assert_array_equal(copy.numpy(), x.numpy())
    np.testing.assert_allclose(n.numpy(), plain, rtol=3 * NORM)
    u = upload(session, stored(rng.standard_normal((3, 200)), "f32"), "f32")
    y, n = A.residual_norm(x, u, post_norm=True)
    np.testing.assert_allclose(y.numpy(), x.numpy() + A.rms_norm(u, -1).numpy(), rtol=3 * NORM, atol=1e-5)
    np.testing.assert_allclose(n.numpy(), A.rms_norm(y, -1).numpy(), rtol=3 * NORM)
    long = upload(session, stored(rng.standard_normal((2, 30000)), "bf16"), "bf16")
    copy, n = A.residual_norm(long, out=(session.empty("bf16", (2, 30000)), session.empty("bf16", (2, 30000))))
    np.testing.assert_array_equal(copy.storage(), long.storage())


def test_infinities_and_nan_stay_in_their_row(session, rng):
    x = rng.standard_normal((3, 600))
    x[1, 77] = np.nan
    y, n = A.residual_norm(upload(session, stored(x, "f32"), "f32"), upload(session, stored(x, "f32"), "f32"))
    assert np.isnan(n.numpy()[1]).all() and np.isfinite(n.numpy()[[0, 2]]).all()
    assert np.isnan(y.numpy()[1]).sum() == 1


@pytest.mark.parametrize("N", [520, 1024, 2000, 4096, 8190, 9000])
def test_many_wide_rows(session, rng, N):
    """As many rows as there are two threads' values of, and one fewer."""
    for M in (511, 512):
        check(session, rng, M, N, post=True, gate="columns", stream="bf16")


def test_more_rows_than_a_grid_holds(session, rng):
    check(session, rng, (1 << 20) + 3, 9, update="bf16", post=True)
