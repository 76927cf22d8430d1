"""Norm weights that a checkpoint does not hold are not taken for ones."""
import numpy as np
import pytest

import affon_amd as A
from affon_amd.decoder import DecoderShape, NORMS, PROJECTIONS, QuantizedDecoderBlock
from tests.test_checkpoint import write_file

pytestmark = pytest.mark.gpu

SHAPE = DecoderShape(width=256, inner_width=512, heads=4, kv_heads=2)


def block_of(session, path, norms):
    entries = []
    for field, module, _, _ in PROJECTIONS:
        out, inp = SHAPE.features(field)
        name = f"model.layers.0.{module}"
        entries += [(name + ".weight", "U32", [out, inp // 4], np.zeros((out, inp // 4), np.uint32).tobytes()),
                    (name + ".scales", "BF16", [out, inp // 64], np.zeros((out, inp // 64), np.uint16).tobytes()),
                    (name + ".biases", "BF16", [out, inp // 64], np.zeros((out, inp // 64), np.uint16).tobytes())]
    entries += [(f"model.layers.0.{NORMS[n]}.weight", "F32", [256], np.ones(256, np.float32).tobytes()) for n in norms]
    path = write_file(path / "block.safetensors", entries, metadata={"format": "mlx"})
    return QuantizedDecoderBlock.from_checkpoint(session, str(path), 0, SHAPE, bits=8, group_size=64)


def step(session, block):
    cache = A.PagedCache(session, pages=1, page_size=16, kv_heads=2, head_dim=64)
    batch = A.DraftBatch(session.tensor(np.zeros((1, 1)), "u32"), session.tensor(np.zeros(1), "u32"), 1)
    return block.step(session.tensor(np.ones((1, 256)), "f32"), None, cache, batch, A.rotary_table(session, 16, 64))


@pytest.mark.parametrize("held", [(), ("attentionNorm",), ("feedForwardNorm",)])
def test_a_checkpoint_without_norms(session, tmp_path, held):
    block = block_of(session, tmp_path, held)
    assert sorted(block.norms) == sorted(held)
    assert len(block.attention(session.empty("bf16", (1, 256)))) == 3
    with pytest.raises(TypeError, match=next(n for n in NORMS if n not in held)):
        step(session, block)


def test_norms_of_ones(session, tmp_path):
    """With both weights, and of a block that is made without any."""
    block = block_of(session, tmp_path, tuple(NORMS))
    made = QuantizedDecoderBlock(SHAPE, block.layers)
    for got in (step(session, block), step(session, made)):
        np.testing.assert_array_equal(got[0].numpy(), np.ones((1, 256)))  # all projections are 0
