"""What appends with head norms and axes, attention over shared prefixes, gathered weights and
eviction refuse, without a GPU: the library checks every descriptor before it looks at the session."""
import ctypes

import pytest

import affon_amd as A
from affon_amd import _native
from tests.test_abi import _view
from tests.test_drafts import BASE, append, attention, batch, cache, refusal

FAR = 1 << 40  # memory of no operand, never read
WEIGHT_BYTES = 2 * 3 * 2 * 64 * 4  # of cache() and batch()


def head_norm(**changes):
    d = dict(query_weight=BASE, key_weight=BASE, query_weight_dtype=_native.BF16, key_weight_dtype=_native.F32,
             epsilon=1e-6, axes=1)
    return _native.HeadNorm(**(d | changes))


def weights(**changes):
    d = dict(query=_view(BASE, (6, 256), (256, 1), _native.BF16), scale=0.1, layer=1, weights=FAR, weights_bytes=WEIGHT_BYTES)
    return _native.WeightsDesc(**(d | changes))


def run_normed(c=None, b=None, d=None, n=None):
    return _native.load().affon_rocm_cache_append_normed(None, c or cache(), b or batch(), d or append(), n or head_norm())


def run_shared(c=None, b=None, d=None, shared=BASE, groups=1):
    return _native.load().affon_rocm_shared_attention(None, c or cache(), b or batch(), d or attention(), shared, groups)


def run_weights(c=None, b=None, d=None):
    return _native.load().affon_rocm_attention_weights(None, c or cache(), b or batch(), d or weights())


def run_evict(c=None, b=None, data=FAR, out=FAR, size=WEIGHT_BYTES, keep=BASE, recent=BASE):
    return _native.load().affon_rocm_cache_evict(None, c or cache(), b or batch(), data, out, size, keep, recent)


def run_commit(c=None, b=None, path=None, accepted=BASE, data=FAR, size=WEIGHT_BYTES):
    path = path or _view(BASE, (3, 2), (2, 1), _native.U32)
    return _native.load().affon_rocm_weights_commit(None, c or cache(), b or batch(), path, accepted, data, size)


RUNS = [run_normed, run_shared, run_weights, run_evict, run_commit]


@pytest.mark.parametrize("run", RUNS)
def test_valid_descriptors_reach_the_session(run):
    assert run() == _native.CORE_FAILURE and "session is not open" in _native.last_error()


@pytest.mark.parametrize("run", RUNS)
@pytest.mark.parametrize("changes,message", [
    ({"dtype": _native.U32}, "f32 or bf16 cache"), ({"layers": 0}, "empty dimension"), ({"page_size": 24}, "multiple of 16"),
    ({"head_dim": 264}, "at most 256"), ({"bytes": 100}, "smaller than its shape"), ({"keys": BASE + 8}, "16-byte aligned")])
def test_caches(run, changes, message):
    assert message in refusal(run(c=cache(**changes)))


@pytest.mark.parametrize("run", RUNS)
def test_batches(run):
    assert "u32 page table" in refusal(run(b=batch(table=_view(BASE, (3, 4), (4, 1), _native.F32))))
    assert "at least one row" in refusal(run(b=batch(rows=0)))
    assert "too many tokens" in refusal(run(b=batch(columns=1 << 27)))
    assert "lengths" in refusal(run(b=batch(lengths=None)))


def test_appends():
    assert "one type" in refusal(run_normed(d=append(key=_view(BASE, (6, 128), (128, 1), _native.BF16))))
    assert "rotary_dim" in refusal(run_normed(d=append(rotary_dim=66)))
    assert "layer" in refusal(run_normed(d=append(layer=2)))
    for changes in ({"query_weight_dtype": _native.U32}, {"key_weight_stride": 1}, {"query_weight_stride": 128},
                    {"query_weight": BASE + 1}, {"key_weight": BASE + 2}):
        assert "norm weights" in refusal(run_normed(n=head_norm(**changes)))
    for epsilon in (0.0, -1.0, float("inf"), float("nan")):
        assert "epsilon" in refusal(run_normed(n=head_norm(epsilon=epsilon)))
    for axes in (0, 5, -1):
        assert "four axes" in refusal(run_normed(n=head_norm(axes=axes)))
    wrong = head_norm(axes=2)
    wrong.axis[31] = 2
    assert "pair has an axis" in refusal(run_normed(n=wrong))
    wrong.axis[31], wrong.axis[32] = 1, 200  # past rotary_dim / 2: not read
    assert run_normed(n=wrong) == _native.CORE_FAILURE
    lib = _native.load()
    refusal(lib.affon_rocm_cache_append_normed(None, cache(), batch(), append(), None))
    refusal(lib.affon_rocm_cache_append_normed(None, cache(), batch(), None, head_norm()))


def test_shared_attentions():
    for changes in ({"shared": None}, {"shared": BASE + 2}, {"groups": 0}, {"groups": -3}, {"groups": 2}, {"groups": 6}):
        assert "groups of equal size" in refusal(run_shared(**changes))
    assert "one type" in refusal(run_shared(d=attention(query=_view(BASE, (6, 256), (256, 1), _native.F32))))
    assert "scale" in refusal(run_shared(d=attention(scale=float("nan"))))
    assert "mask must be [6, 1]" in refusal(run_shared(d=attention(mask=_view(BASE, (5, 1), (1, 1), _native.U32))))
    assert "output buffer" in refusal(run_shared(d=attention(output=None)))
    assert "layer" in refusal(run_shared(d=attention(layer=-1)))
    refusal(_native.load().affon_rocm_shared_attention(None, cache(), batch(), None, BASE, 1))


def test_gathered_weights():
    for changes in ({"weights": None}, {"weights": FAR + 2}, {"weights_bytes": WEIGHT_BYTES - 1}):
        assert "f32 weights" in refusal(run_weights(d=weights(**changes)))
    assert "multiple of kv_heads" in refusal(run_weights(d=weights(query=_view(BASE, (6, 192), (192, 1), _native.BF16))))
    assert "scale" in refusal(run_weights(d=weights(scale=float("inf"))))
    assert "layer" in refusal(run_weights(d=weights(layer=2)))
    refusal(_native.load().affon_rocm_attention_weights(None, cache(), batch(), None))


def test_evictions():
    for changes in ({"data": None}, {"out": None}, {"data": FAR + 1}, {"size": WEIGHT_BYTES - 4}):
        assert "f32 weights" in refusal(run_evict(**changes))
    for changes in ({"keep": None}, {"recent": None}, {"keep": BASE + 1}, {"recent": BASE + 3}):
        assert "tokens to keep" in refusal(run_evict(**changes))


def test_commits():
    assert "at most the batch's rows" in refusal(run_commit(path=_view(BASE, (3, 3), (3, 1), _native.U32)))
    assert "accepted" in refusal(run_commit(accepted=None))
    assert "f32 weights" in refusal(run_commit(size=0))


def test_axes():
    for sections, message in (((), "one to four"), ((1, 2, 3, 4, 5), "one to four"), ((0, 4), "positive"), ((2.0, 2), "positive"),
                              ((100, 29), "at most 128")):
        with pytest.raises(TypeError, match=message):
            A.rotary_axes(sections)
    for axes in ((), (4,), (-1,), (0,) * 129, (0.0,), (True,)):
        with pytest.raises(TypeError, match="1 to 128 axes"):
            A.RotaryAxes(axes)
    assert A.rotary_axes((1, 2)).axes == (0, 1, 1) and A.rotary_axes([2, 1], interleaved=True).axes == (0, 1, 0)


def test_structures_have_the_sizes_of_the_header():
    """A pair's axes lie behind three words of strides and types, as in C."""
    assert ctypes.sizeof(_native.HeadNorm) == 4 * 8 + 4 * 4 + 128 and _native.HeadNorm.axis.offset == 48
    assert ctypes.sizeof(_native.WeightsDesc) == 2 * ctypes.sizeof(_native.View) + 4 * 8
