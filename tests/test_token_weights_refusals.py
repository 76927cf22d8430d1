"""What token_weights refuses, without a GPU."""
import pytest

from affon_amd import _native
from tests.test_cache_refusals import FAR, WEIGHT_BYTES
from tests.test_drafts import BASE, batch, cache, refusal


def run(c=None, b=None, data=FAR, size=WEIGHT_BYTES):
    return _native.load().affon_rocm_token_weights(None, c or cache(), b or batch(), data, size)


def test_a_valid_call_reaches_the_session():
    assert run() == _native.CORE_FAILURE and "session is not open" in _native.last_error()


@pytest.mark.parametrize("changes", [{"data": None}, {"data": FAR + 2}, {"size": WEIGHT_BYTES - 1}, {"size": 0}])
def test_weights(changes):
    assert "f32 weights" in refusal(run(**changes))


def test_caches_and_batches():
    assert "16-byte aligned" in refusal(run(c=cache(keys=BASE + 8)))
    assert "multiple of 16" in refusal(run(c=cache(page_size=24)))
    refusal(run(b=batch(rows=0)))
    refusal(run(b=batch(lengths=None)))
