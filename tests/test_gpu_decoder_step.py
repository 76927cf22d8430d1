"""A decoder block over drafted tokens: the projections' Programs with the
norms, the cache and the attention between them.

Against the formulas in 64 bits on the device's own projections the bound is
rtol 2e-2 with atol 2e-2 of the root mean square: two roundings to bf16 (the
normalized stream and the attention's result) before projections that the
framework's tests hold to rtol 1e-2 each. Token by token against all at once
the same sums run through other kernels and orders: the same bound."""
import numpy as np
import pytest

import affon_amd as A
from affon_amd.decoder import DecoderShape, NORMS, PROJECTIONS, QuantizedDecoderBlock
from oracle import oracle as O
from tests.drafts import mask_words, set_tensor, stored, tree, upload, widened
from tests.test_checkpoint import write_file

pytestmark = pytest.mark.gpu

SHAPE = DecoderShape(width=256, inner_width=512, heads=4, kv_heads=2)
BITS, GROUP, PAGE, BLOCKS = 8, 64, 16, 2


def close(got, want):
    got, want = got.astype(np.float64), np.asarray(want, np.float64)
    rms = np.sqrt(np.mean(want ** 2))
    assert (np.abs(got - want) <= 2e-2 * np.abs(want) + 2e-2 * rms).all(), float(np.abs(got - want).max() / rms)


@pytest.fixture(scope="module")
def blocks(session, tmp_path_factory):
    """Two blocks of a checkpoint, and their weights in f64."""
    entries, arrays, rng = [], [], np.random.default_rng(5)
    for index in range(BLOCKS):
        arrays.append({})
        for field, module, _, _ in PROJECTIONS:
            out, inp = SHAPE.features(field)
            packed, s, b = O.quantize(stored(rng.standard_normal((out, inp)) * 0.05, "bf16"), BITS, GROUP, "bf16")
            arrays[-1][field] = O.dequantize(packed, s, b, BITS, GROUP, "f32").astype(np.float64)
            name = f"model.layers.{index}.{module}"
            entries += [(name + ".weight", "U32", list(packed.shape), packed.tobytes()),
                        (name + ".scales", "BF16", list(s.shape), s.tobytes()),
                        (name + ".biases", "BF16", list(b.shape), b.tobytes())]
        for field, module in NORMS.items():
            weight = stored(1 + 0.2 * rng.standard_normal(SHAPE.width), "bf16")
            arrays[-1][field] = widened(weight)
            entries.append((f"model.layers.{index}.{module}.weight", "BF16", [SHAPE.width], weight.tobytes()))
    path = write_file(tmp_path_factory.mktemp("step") / "blocks.safetensors", entries, metadata={"format": "mlx"})
    built = [QuantizedDecoderBlock.from_checkpoint(session, str(path), i, SHAPE, bits=BITS, group_size=GROUP)
             for i in range(BLOCKS)]
    assert all(sorted(b.norms) == sorted(NORMS) for b in built)
    return built, arrays


class Model:
    """The blocks over a cache of two sequences, and the step of a batch."""

    def __init__(self, session, blocks, T, lengths=(0, 0)):
        self.session, self.blocks = session, blocks
        self.cache = A.PagedCache(session, pages=12, page_size=PAGE, kv_heads=2, head_dim=64, layers=BLOCKS)
        self.table = upload(session, np.array([[3, 7, 1, 5], [0, 9, 2, 11]], np.uint32), "u32")
        self.lengths = upload(session, np.array(lengths, np.uint32), "u32")
        self.rotary = A.rotary_table(session, 64, 64)
        self.T = T

    def run(self, x, mask=None, depth=None, T=None):
        T = T or self.T
        batch = A.DraftBatch(self.table, self.lengths, T)
        lengths = self.lengths.numpy().astype(np.int64)
        if depth is not None:
            depth = upload(self.session, (depth + lengths[:, None]).reshape(-1).astype(np.uint32), "u32")
        if mask is not None:
            mask = upload(self.session, mask_words(mask), "u32")
        stream, update = upload(self.session, x.astype(np.float32), "f32"), None
        for i, block in enumerate(self.blocks):
            stream, update = block.step(stream, update, self.cache, batch, self.rotary, positions=depth, mask=mask,
                                        layer=i)
        return A.residual_norm(stream, update)[1].numpy()

    def grow(self, by):
        set_tensor(self.lengths, self.lengths.numpy() + np.asarray(by, np.uint32))


def expected(x, arrays, positions, sees):
    """The blocks in f64: x [n, width] of one sequence, token i seeing those of sees[i]."""
    norm = lambda v, w: v / np.sqrt((v ** 2).mean(-1, keepdims=True) + 1e-5) * w
    angle = np.outer(positions, 10000.0 ** (-np.arange(32) / 32))
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    turn = lambda v: np.concatenate([v[..., :32] * c - v[..., 32:] * s, v[..., 32:] * c + v[..., :32] * s], -1)
    for w in arrays:
        n = norm(x, w["attentionNorm"])
        q, k, v = (n @ w[name].T for name in ("query", "key", "value"))
        q, k, v = turn(q.reshape(len(x), 4, 64)), turn(k.reshape(len(x), 2, 64)), v.reshape(len(x), 2, 64)
        out = np.zeros((len(x), 4, 64))
        for i in range(len(x)):
            for h in range(4):
                score = k[sees[i], h // 2] @ q[i, h] / 8.0
                p = np.exp(score - score.max())
                out[i, h] = p / p.sum() @ v[sees[i], h // 2]
        x = x + out.reshape(len(x), -1) @ w["attentionOutput"].T
        n = norm(x, w["feedForwardNorm"])
        gate = n @ w["gate"].T
        x = x + (gate / (1 + np.exp(-gate)) * (n @ w["up"].T)) @ w["down"].T
    return norm(x, 1.0)


def test_a_tree_after_a_prompt(session, blocks, rng):
    built, arrays = blocks
    prompt, drafts = rng.standard_normal((2, 20, 256)), rng.standard_normal((2, 7, 256))
    model = Model(session, built, 20)
    got = model.run(prompt.reshape(-1, 256)).reshape(2, 20, 256)
    for b in range(2):
        close(got[b], expected(prompt[b], arrays, np.arange(20), [np.arange(i + 1) for i in range(20)]))
    model.grow([20, 20])
    mask = tree(rng, 2, 7)
    depth = mask.sum(1).reshape(2, 7) - 1
    got = model.run(drafts.reshape(-1, 256), mask, depth, T=7).reshape(2, 7, 256)
    for b in range(2):
        sees = [np.arange(i + 1) for i in range(20)] + [
            np.concatenate([np.arange(20), 20 + np.nonzero(mask[b * 7 + i])[0]]) for i in range(7)]
        want = expected(np.concatenate([prompt[b], drafts[b]]), arrays, np.concatenate([np.arange(20), 20 + depth[b]]), sees)
        close(got[b], want[20:])


def test_accepted_tokens_go_on_as_if_they_came_one_by_one(session, blocks, rng):
    """A tree, its accepted path committed, and a next token: as the path's
    tokens one at a time, and that token."""
    built, _ = blocks
    first, drafts, last = rng.standard_normal((2, 3, 256)), rng.standard_normal((2, 6, 256)), rng.standard_normal((2, 256))
    parents = np.array([[-1, 0, 0, 1, 2, 4], [-1, 0, 1, 1, 3, 0]])
    paths, accepted = np.array([[0, 2, 4, 5], [0, 1, 3, 0]], np.uint32), np.array([4, 3], np.uint32)
    mask = np.zeros((2, 6, 6), bool)
    for b in range(2):
        for i in range(6):
            if i:
                mask[b, i] = mask[b, parents[b, i]]
            mask[b, i, i] = True
    model = Model(session, built, 3)
    model.run(first.reshape(-1, 256))
    model.grow([3, 3])
    all_at_once = model.run(drafts.reshape(-1, 256), mask.reshape(12, 6), mask.sum(-1) - 1, T=6).reshape(2, 6, 256)
    A.cache_commit(model.cache, A.DraftBatch(model.table, model.lengths, 6), upload(session, paths, "u32"),
                   upload(session, accepted, "u32"))
    model.grow(accepted)
    next_token = model.run(last, T=1)

    single = Model(session, built, 3)
    single.run(first.reshape(-1, 256))
    single.grow([3, 3])
    for i in range(4):
        got = single.run(np.stack([drafts[b, paths[b, i]] for b in range(2)]), T=1)
        for b in range(2):
            if i < accepted[b]:
                close(all_at_once[b, paths[b, i]], got[b])
        single.grow((i < accepted).astype(np.uint32))
    close(next_token, single.run(last, T=1))


def test_norm_weights_of_other_shapes(session, tmp_path):
    """They are not read; the projections are, and a step refuses."""
    entries = []
    for field, module, _, _ in PROJECTIONS:
        out, inp = SHAPE.features(field)
        name = f"model.layers.0.{module}"
        entries += [(name + ".weight", "U32", [out, inp // 4], np.zeros((out, inp // 4), np.uint32).tobytes()),
                    (name + ".scales", "BF16", [out, inp // GROUP], np.zeros((out, inp // GROUP), np.uint16).tobytes()),
                    (name + ".biases", "BF16", [out, inp // GROUP], np.zeros((out, inp // GROUP), np.uint16).tobytes())]
    entries.append(("model.layers.0.input_layernorm.weight", "F32", [1, 256], np.ones(256, np.float32).tobytes()))
    path = write_file(tmp_path / "block.safetensors", entries, metadata={"format": "mlx"})
    block = QuantizedDecoderBlock.from_checkpoint(session, str(path), 0, SHAPE, bits=BITS, group_size=GROUP)
    assert not block.norms and len(block.attention(session.empty("bf16", (1, 256)))) == 3
    model = Model(session, [block], 1)
    with pytest.raises(TypeError, match="attentionNorm"):
        model.run(np.zeros((2, 256)))


def test_what_a_block_refuses(blocks):
    built, _ = blocks
    block = built[0]
    with pytest.raises(TypeError, match="unknown norm"):
        QuantizedDecoderBlock(SHAPE, block.layers, norms={"other": block.norms["attentionNorm"]})
    with pytest.raises(TypeError, match="attentionNorm must be"):
        QuantizedDecoderBlock(SHAPE, block.layers, norms={"attentionNorm": block.layers["gate"].scales})
