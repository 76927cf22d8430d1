"""What the drafted-token ops and residual_norm refuse, without a GPU: the
library checks every descriptor before it looks at the session."""
import numpy as np
import pytest

from affon_amd import _native
from tests.drafts import mask_words, tree
from tests.test_abi import _view

BASE = 1 << 20  # an address that is never read


def cache(**changes):
    c = dict(keys=BASE, values=2 * BASE, layers=2, pages=5, kv_heads=2, page_size=16, head_dim=64, dtype=_native.BF16)
    c |= changes
    size = 4 if c["dtype"] == _native.F32 else 2
    c.setdefault("bytes", max(0, c["layers"] * c["pages"] * c["kv_heads"] * c["page_size"] * c["head_dim"] * size))
    return _native.KvCache(**c)


def batch(B=3, columns=4, rows=2, lengths=BASE, counts=None, table=None):
    view = table if table is not None else _view(BASE, (B, columns), (columns, 1), _native.U32)
    return _native.DraftBatch(view, lengths, counts, rows)


def append(**changes):
    d = dict(query=_view(BASE, (6, 256), (256, 1), _native.F32), key=_view(BASE, (6, 128), (128, 1), _native.F32),
             value=_view(BASE, (6, 128), (128, 1), _native.F32), positions=None, rotary=BASE, rotary_rows=9,
             rotary_dim=64, interleaved=0, layer=1, output=BASE, output_bytes=6 * 256 * 2)
    return _native.AppendDesc(**(d | changes))


def attention(**changes):
    d = dict(query=_view(BASE, (6, 256), (256, 1), _native.BF16), scale=0.1, layer=0, output=BASE,
             output_bytes=6 * 256 * 2)
    return _native.AttentionDesc(**(d | changes))


def norm(**changes):
    d = dict(stream=BASE, update=BASE, stream_out=BASE, normalized=BASE, rows=3, cols=10, stream_stride=10,
             update_stride=10, stream_out_stride=10, normalized_stride=10, scale=1.0, epsilon=1e-5)
    return _native.ResidualNormDesc(**(d | changes))


def refusal(status):
    assert status == _native.INVALID_SHAPE, (status, _native.last_error())
    return _native.last_error()


def run_append(c=None, b=None, d=None):
    return _native.load().affon_rocm_cache_append(None, c or cache(), b or batch(), d or append())


def run_attention(c=None, b=None, d=None):
    return _native.load().affon_rocm_tree_attention(None, c or cache(), b or batch(), d or attention())


def run_commit(c=None, b=None, path=None, accepted=BASE):
    path = path or _view(BASE, (3, 2), (2, 1), _native.U32)
    return _native.load().affon_rocm_cache_commit(None, c or cache(), b or batch(), path, accepted)


def test_valid_descriptors_reach_the_session():
    lib = _native.load()
    f32 = dict(c=cache(dtype=_native.F32),
               d=attention(query=_view(BASE, (6, 256), (300, 1), _native.F32), output_bytes=6 * 256 * 4))
    for status in (run_append(), run_attention(), run_attention(**f32), run_commit(),
                   lib.affon_rocm_residual_norm(None, norm()),
                   lib.affon_rocm_residual_norm(None, norm(update=None, stream_out=None, stream_stride=0))):
        assert status == _native.CORE_FAILURE and "session is not open" in _native.last_error()


@pytest.mark.parametrize("run", [run_append, run_attention, run_commit])
@pytest.mark.parametrize("changes,message", [
    ({"dtype": _native.U32}, "f32 or bf16 cache"), ({"layers": 0}, "empty dimension"), ({"pages": -1}, "empty dimension"),
    ({"pages": 1 << 39}, "overflows"), ({"page_size": 24}, "multiple of 16"), ({"head_dim": 60}, "multiple of 8"),
    ({"head_dim": 264}, "at most 256"), ({"bytes": 100}, "smaller than its shape"), ({"values": None}, "smaller"),
    ({"keys": BASE + 8}, "16-byte aligned")])
def test_caches(run, changes, message):
    assert message in refusal(run(c=cache(**changes)))


@pytest.mark.parametrize("run", [run_append, run_attention, run_commit])
def test_batches(run):
    assert "u32 page table" in refusal(run(b=batch(table=_view(BASE, (3, 4), (4, 1), _native.F32))))
    assert "unit inner stride" in refusal(run(b=batch(table=_view(BASE, (3, 4), (8, 2), _native.U32))))
    assert "exceeds its buffer" in refusal(run(b=batch(table=_view(BASE, (3, 4), (4, 1), _native.U32, buffer_bytes=40))))
    assert "at least one row" in refusal(run(b=batch(rows=0)))
    assert "at least one row" in refusal(run(b=batch(rows=1 << 30)))
    assert "too many tokens" in refusal(run(b=batch(columns=1 << 27)))
    assert "lengths" in refusal(run(b=batch(lengths=None)))
    assert "lengths" in refusal(run(b=batch(counts=BASE + 2)))


def test_appends():
    wrong = _view(BASE, (6, 120), (120, 1), _native.F32)
    assert "one type" in refusal(run_append(d=append(key=_view(BASE, (6, 128), (128, 1), _native.BF16))))
    assert "multiple of kv_heads" in refusal(run_append(d=append(query=_view(BASE, (6, 192), (192, 1), _native.F32))))
    assert "query must be [6, 256]" in refusal(run_append(d=append(query=_view(BASE, (5, 256), (256, 1), _native.F32))))
    assert "key must be [6, 128]" in refusal(run_append(d=append(key=wrong)))
    assert "value must be [6, 128]" in refusal(run_append(d=append(value=wrong)))
    assert "element aligned" in refusal(run_append(d=append(value=_view(BASE + 2, (6, 128), (128, 1), _native.F32))))
    for dim in (0, 7, 66):
        assert "rotary_dim" in refusal(run_append(d=append(rotary_dim=dim)))
    assert "rotary table" in refusal(run_append(d=append(rotary=None)))
    assert "rotary table" in refusal(run_append(d=append(rotary_rows=0)))
    assert "output buffer" in refusal(run_append(d=append(output_bytes=6 * 256 * 2 - 1)))
    for layer in (-1, 2):
        assert "layer" in refusal(run_append(d=append(layer=layer)))


def test_attentions():
    assert "one type" in refusal(run_attention(d=attention(query=_view(BASE, (6, 256), (256, 1), _native.F32))))
    for scale in (float("nan"), float("inf")):
        assert "scale" in refusal(run_attention(d=attention(scale=scale)))
    assert "bit for every row" in refusal(run_attention(b=batch(B=1, rows=33), d=attention(
        query=_view(BASE, (33, 256), (256, 1), _native.BF16), output_bytes=33 * 512,
        mask=_view(BASE, (33, 1), (1, 1), _native.U32))))
    assert "mask must be [6, 1]" in refusal(run_attention(d=attention(mask=_view(BASE, (5, 1), (1, 1), _native.U32))))
    assert "u32 mask" in refusal(run_attention(d=attention(mask=_view(BASE, (6, 1), (1, 1), _native.F32))))
    assert "layer" in refusal(run_attention(d=attention(layer=5)))


def test_commits():
    assert "at most the batch's rows" in refusal(run_commit(path=_view(BASE, (3, 3), (3, 1), _native.U32)))
    assert "path must be [3, 2]" in refusal(run_commit(path=_view(BASE, (2, 2), (2, 1), _native.U32)))
    assert "u32 path" in refusal(run_commit(path=_view(BASE, (3, 2), (2, 1), _native.F32)))
    assert "accepted" in refusal(run_commit(accepted=None))


def test_norms():
    run = lambda **changes: refusal(_native.load().affon_rocm_residual_norm(None, norm(**changes)))
    assert "f32 or bf16" in run(stream_dtype=_native.U32)
    assert "non-empty" in run(rows=0) and "non-empty" in run(cols=-5) and "non-empty" in run(cols=1 << 29)
    assert "null" in run(stream=None) and "null" in run(normalized=None) and "null" in run(stream_out=None)
    assert "no gate" in run(update=None, gate=BASE) and "no post_norm" in run(update=None, post_norm=1)
    assert "needs post_norm" in run(post_weight=BASE)
    assert "aligned" in run(update=BASE + 2) and "aligned" in run(weight=BASE + 1, weight_dtype=_native.BF16)
    assert "row stride" in run(stream_out_stride=9) and "row stride" in run(update_stride=-1)
    for epsilon in (0.0, -1.0, float("inf"), float("nan")):
        assert "epsilon" in run(epsilon=epsilon)
    assert "scale" in run(scale=float("inf"))


def test_null_descriptors():
    lib = _native.load()
    for status in (lib.affon_rocm_cache_append(None, None, batch(), append()),
                   lib.affon_rocm_cache_append(None, cache(), None, append()),
                   lib.affon_rocm_cache_append(None, cache(), batch(), None),
                   lib.affon_rocm_tree_attention(None, cache(), batch(), None),
                   lib.affon_rocm_cache_commit(None, cache(), batch(), None, BASE),
                   lib.affon_rocm_residual_norm(None, None)):
        refusal(status)


def test_mask_words_hold_the_bits_of_the_mask():
    mask = tree(np.random.default_rng(3), 2, 45)
    words = mask_words(mask)
    assert words.shape == (90, 2)
    for r, j in ((0, 0), (44, 44), (60, 3), (89, 33)):
        assert bool(words[r, j // 32] >> (j % 32) & 1) == mask[r, j]
