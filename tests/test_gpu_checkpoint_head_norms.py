"""Which of a checkpoint's query and key norms a decoder block reads."""
import numpy as np
import pytest

from affon_amd.decoder import QuantizedDecoderBlock
from tests.test_gpu_decoder_serving import Server, checkpoint, expected
from tests.test_gpu_decoder_step import BITS, GROUP, SHAPE, close

pytestmark = pytest.mark.gpu


def load(session, path, **options):
    return [QuantizedDecoderBlock.from_checkpoint(session, str(path), i, SHAPE, bits=BITS, group_size=GROUP, **options)
            for i in range(2)]


def run(session, blocks, arrays, rng, normed):
    x = rng.standard_normal((1, 9, 256))
    got = Server(session, blocks, 1).run(x, 9)
    close(got[0], expected(x[0], arrays, np.arange(9)[None], [np.arange(i + 1) for i in range(9)], [0] * 32, normed=normed))


def test_norms_that_are_there_are_read(session, rng, tmp_path):
    arrays = checkpoint(tmp_path / "blocks.safetensors", rng)
    blocks = load(session, tmp_path / "blocks.safetensors")
    assert [sorted(b.head_norms) for b in blocks] == [["keyNorm", "queryNorm"]] * 2
    run(session, blocks, arrays, rng, True)


def test_without_norms(session, rng, tmp_path):
    arrays = checkpoint(tmp_path / "blocks.safetensors", rng, leave_out=("queryNorm", "keyNorm"))
    blocks = load(session, tmp_path / "blocks.safetensors")
    assert all(not b.head_norms and not b.unread_norms for b in blocks)
    run(session, blocks, arrays, rng, False)
    assert load(session, tmp_path / "blocks.safetensors", head_norms=True)[0].unread_norms == ("queryNorm", "keyNorm")


def test_a_norm_of_one_kind(session, tmp_path):
    checkpoint(tmp_path / "blocks.safetensors", np.random.default_rng(2), leave_out=("keyNorm",))
    block = load(session, tmp_path / "blocks.safetensors")[0]
    assert sorted(block.head_norms) == ["queryNorm"] and block.unread_norms == ()


def test_a_norm_that_cannot_be_read(session, tmp_path):
    checkpoint(tmp_path / "blocks.safetensors", np.random.default_rng(3), head_shapes={"keyNorm": 32})
    blocks = load(session, tmp_path / "blocks.safetensors")
    assert blocks[0].unread_norms == ("keyNorm",)
    with pytest.raises(TypeError, match="keyNorm"):
        Server(session, blocks, 1).run(np.zeros((1, 1, 256)), 1)


def test_each_heads_own_weights_or_a_wider_norm(session, rng, tmp_path):
    """The file does not tell them apart: taken for each head's own where the caller says so."""
    arrays = checkpoint(tmp_path / "blocks.safetensors", rng, head_shapes={"queryNorm": 256, "keyNorm": 128})
    blocks = load(session, tmp_path / "blocks.safetensors")
    assert blocks[0].unread_norms == ("queryNorm", "keyNorm")
    with pytest.raises(TypeError, match="queryNorm, keyNorm.*head_norms=True"):
        Server(session, blocks, 1).run(np.zeros((1, 1, 256)), 1)
    run(session, load(session, tmp_path / "blocks.safetensors", head_norms=True), arrays, rng, True)


def test_norms_that_are_left_out(session, rng, tmp_path):
    """Asked for: the step is the plain one."""
    arrays = checkpoint(tmp_path / "blocks.safetensors", rng)
    blocks = load(session, tmp_path / "blocks.safetensors", head_norms=False)
    assert all(not b.head_norms and not b.unread_norms for b in blocks)
    run(session, blocks, arrays, rng, False)
