"""A decoder block's step with head norms, positions of several axes, shared
prefixes and gathered weights, one after the other as a server uses them.

Bounds as in the tests of the plain step: against 64 bits on the device's own
projections rtol 2e-2 with atol 2e-2 of the root mean square, and the same
between two orders of the same sums."""
import numpy as np
import pytest

import affon_amd as A
from affon_amd.decoder import HEAD_NORMS, NORMS, PROJECTIONS, QuantizedDecoderBlock
from oracle import oracle as O
from tests.drafts import mask_words, stored, tree, upload, widened
from tests.test_checkpoint import write_file
from tests.test_gpu_decoder_step import BITS, GROUP, PAGE, SHAPE, close

pytestmark = pytest.mark.gpu


def checkpoint(path, rng, blocks=2, leave_out=(), head_shapes=None):
    entries, arrays = [], []
    for index in range(blocks):
        arrays.append({})
        for field, module, _, _ in PROJECTIONS:
            out, inp = SHAPE.features(field)
            packed, s, b = O.quantize(stored(rng.standard_normal((out, inp)) * 0.05, "bf16"), BITS, GROUP, "bf16")
            arrays[-1][field] = O.dequantize(packed, s, b, BITS, GROUP, "f32").astype(np.float64)
            name = f"model.layers.{index}.{module}"
            entries += [(name + ".weight", "U32", list(packed.shape), packed.tobytes()),
                        (name + ".scales", "BF16", list(s.shape), s.tobytes()),
                        (name + ".biases", "BF16", list(b.shape), b.tobytes())]
        for field, module in (NORMS | HEAD_NORMS).items():
            if field in leave_out:
                continue
            size = SHAPE.width if field in NORMS else (head_shapes or {}).get(field, 64)
            weight = stored(1 + 0.2 * rng.standard_normal(size), "bf16")
            arrays[-1][field] = widened(weight)
            entries.append((f"model.layers.{index}.{module}.weight", "BF16", [size], weight.tobytes()))
    write_file(path, entries, metadata={"format": "mlx"})
    return arrays


def load(session, path, **options):
    return [QuantizedDecoderBlock.from_checkpoint(session, str(path), i, SHAPE, bits=BITS, group_size=GROUP,
                                                  **({"head_norms": True} | options)) for i in range(2)]


@pytest.fixture(scope="module")
def model(session, tmp_path_factory):
    path = tmp_path_factory.mktemp("serving") / "blocks.safetensors"
    arrays = checkpoint(path, np.random.default_rng(11), head_shapes={"queryNorm": 256})
    return load(session, path), arrays


def expected(x, arrays, positions, sees, axes, normed=True):
    """Blocks in f64: x [n, width] of one sequence, positions [axes, n], token i seeing those of sees[i]."""
    norm = lambda v, w: v / np.sqrt((v ** 2).mean(-1, keepdims=True) + 1e-5) * w
    angle = np.asarray(positions, np.float64)[axes].T * 10000.0 ** (-np.arange(32) / 32)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    turn = lambda v: np.concatenate([v[..., :32] * c - v[..., 32:] * s, v[..., 32:] * c + v[..., :32] * s], -1)
    for w in arrays:
        n = norm(x, w["attentionNorm"])
        q, k, v = (n @ w[name].T for name in ("query", "key", "value"))
        q, k, v = q.reshape(len(x), 4, 64), k.reshape(len(x), 2, 64), v.reshape(len(x), 2, 64)
        if normed:
            q, k = norm(q, w["queryNorm"].reshape(-1, 64)), norm(k, w["keyNorm"].reshape(-1, 64))
        q, k = turn(q), turn(k)
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


class Server:
    """Blocks over a cache of B sequences, each with its own pages but for those of a shared prefix."""

    def __init__(self, session, blocks, B, columns=8, prefix_pages=0):
        self.session, self.blocks, self.B = session, blocks, B
        own = columns - prefix_pages
        table = np.zeros((B, columns), np.uint32)
        table[:, :prefix_pages] = np.arange(prefix_pages)
        table[:, prefix_pages:] = prefix_pages + np.arange(B * own).reshape(B, own)
        self.cache = A.PagedCache(session, pages=prefix_pages + B * own, page_size=PAGE, kv_heads=2, head_dim=64, layers=2)
        self.table = upload(session, table, "u32")
        self.lengths = upload(session, np.zeros(B, np.uint32), "u32")
        self.rotary = A.rotary_table(session, 256, 64)

    def run(self, x, T, mask=None, positions=None, **options):
        batch = A.DraftBatch(self.table, self.lengths, T)
        stream, update = upload(self.session, x.reshape(self.B * T, -1).astype(np.float32), "f32"), None
        if positions is not None:
            positions = upload(self.session, np.asarray(positions, np.uint32), "u32")
        if mask is not None:
            mask = upload(self.session, mask_words(mask), "u32")
        for i, block in enumerate(self.blocks):
            stream, update = block.step(stream, update, self.cache, batch, self.rotary, positions=positions, mask=mask,
                                        layer=i, **options)
        return A.residual_norm(stream, update)[1].numpy().reshape(self.B, T, -1)

    def grow(self, by):
        self.lengths.write(self.lengths.numpy() + np.asarray(by, np.uint32))


def test_head_norms_and_axes(session, model, rng):
    """A text, then an image of 3 x 4 patches with positions of time, height and width."""
    blocks, arrays = model
    axes = A.rotary_axes((8, 12, 12))
    server = Server(session, blocks, 2)
    text, image = rng.standard_normal((2, 5, 256)), rng.standard_normal((2, 12, 256))
    first = np.tile(np.arange(5), (3, 1))
    then = 5 + np.stack([np.zeros(12, int), np.arange(12) // 4, np.arange(12) % 4])
    got = server.run(text, 5, positions=np.tile(first, (1, 2)), axes=axes)
    server.grow(5)
    image_got = server.run(image, 12, positions=np.tile(then, (1, 2)), axes=axes)
    for b in range(2):
        want = expected(np.concatenate([text[b], image[b]]), arrays, np.concatenate([first, then], 1),
                        [np.arange(i + 1) for i in range(17)], list(axes.axes))
        close(got[b], want[:5])
        close(image_got[b], want[5:])


def test_a_shared_prompt(session, model, rng):
    """One prompt's pages under four samples: a tree of drafted tokens, committed, and a next token,
    as with tree_attention over each sequence's own copy."""
    blocks, arrays = model
    prompt = rng.standard_normal((1, 96, 256))
    servers = {}
    for name in ("shared", "own"):
        server = Server(session, blocks, 4, columns=10, prefix_pages=6 if name == "shared" else 0)
        server.run(np.repeat(prompt, 4, 0), 96)  # all write the same prompt, the shared pages four times over
        server.grow(96)
        servers[name] = server
    shared = upload(session, np.array([96], np.uint32), "u32")
    drafts, mask = rng.standard_normal((4, 5, 256)), tree(rng, 4, 5)
    depth = 96 + mask.sum(1) - 1
    got = servers["shared"].run(drafts, 5, mask, depth, shared=shared)
    close(got, servers["own"].run(drafts, 5, mask, depth))
    sees = [np.arange(i + 1) for i in range(96)]
    for b in range(4):
        rows = [np.concatenate([np.arange(96), 96 + np.nonzero(mask[b * 5 + i])[0]]) for i in range(5)]
        want = expected(np.concatenate([prompt[0], drafts[b]]), arrays, np.concatenate([np.arange(96), depth[b * 5:b * 5 + 5]])[None],
                        sees + rows, [0] * 32)
        close(got[b], want[96:])
    path, accepted = np.array([[0, 1], [0, 0], [0, 3], [0, 4]], np.uint32), np.array([1, 1, 2, 2], np.uint32)
    mask2 = mask.reshape(4, 5, 5)
    accepted[2:] = [1 + bool(mask2[2, 3, 0]), 1 + bool(mask2[3, 4, 0])]
    for server in servers.values():
        A.cache_commit(server.cache, A.DraftBatch(server.table, server.lengths, 5), upload(session, path, "u32"),
                       upload(session, accepted, "u32"))
        server.grow(accepted)
    last = rng.standard_normal((4, 1, 256))
    close(servers["shared"].run(last, 1, shared=shared), servers["own"].run(last, 1))


def test_a_cache_below_a_budget(session, model, rng):
    """A prompt whose weights are gathered, evictions every few tokens, and steps over what is left: as the
    formula over the tokens that each key head has kept."""
    blocks, _ = model
    server = Server(session, blocks, 2)
    batch = A.DraftBatch(server.table, server.lengths, 1)
    weights = A.token_weights(server.cache, batch)
    server.run(rng.standard_normal((2, 60, 256)), 60, weights=weights)
    server.grow(60)
    first = weights.numpy()
    # Every row's probabilities sum to 1: two heads to a key head.
    np.testing.assert_allclose(first[..., :60].sum(-1), 60 * 2, rtol=1e-5)
    assert not first[..., 60:].any()
    keep, recent = (upload(session, np.array(v, np.uint32), "u32") for v in ([40, 48], [16, 16]))
    place = 60
    for _ in range(3):
        A.cache_evict(server.cache, batch, weights, keep, recent, out=weights)
        server.lengths.write(np.minimum(server.lengths.numpy(), keep.numpy()))
        for _ in range(4):
            before = weights.numpy()
            lengths = server.lengths.numpy().astype(int)
            server.run(rng.standard_normal((2, 1, 256)), 1, positions=[place, place], weights=weights)
            after = weights.numpy()
            for b in range(2):
                grown = after[:, b, :, :lengths[b] + 1].sum(-1) - before[:, b, :, :lengths[b]].sum(-1)
                np.testing.assert_allclose(grown, 2.0, rtol=1e-4)  # a difference of sums of about 120, in f32
            server.grow(1)
            place += 1
    assert list(server.lengths.numpy()) == [44, 52]


def test_steps_without_the_options_are_as_before(session, model, rng):
    """head_norms off: the checkpoint's head norms are not read, and the step is the plain one."""
    blocks, arrays = model
    plain = [QuantizedDecoderBlock(SHAPE, b.layers, norms=b.norms) for b in blocks]
    x = rng.standard_normal((1, 9, 256))
    got = Server(session, plain, 1).run(x, 9)
    close(got[0], expected(x[0], arrays, np.arange(9)[None], [np.arange(i + 1) for i in range(9)], [0] * 32, normed=False))


def test_what_a_block_refuses(session, model, tmp_path):
    blocks, _ = model
    layers, norms = blocks[0].layers, blocks[0].norms
    with pytest.raises(TypeError, match="unknown head norm"):
        QuantizedDecoderBlock(SHAPE, layers, head_norms={"valueNorm": norms["attentionNorm"]})
    with pytest.raises(TypeError, match="keyNorm must be"):
        QuantizedDecoderBlock(SHAPE, layers, head_norms={"keyNorm": norms["attentionNorm"]})
    for leave_out, shapes in ((("keyNorm",), None), ((), {"keyNorm": 32})):
        checkpoint(tmp_path / "blocks.safetensors", np.random.default_rng(1), leave_out=leave_out, head_shapes=shapes)
        found = load(session, tmp_path / "blocks.safetensors")
        assert found[0].unread_norms == ("keyNorm",)
        with pytest.raises(TypeError, match="keyNorm"):
            Server(session, found, 1).run(np.zeros((1, 1, 256)), 1)
        assert load(session, tmp_path / "blocks.safetensors", head_norms=False)[0].unread_norms == ()
