"""Quantized projections of a Llama-style decoder block, authored as Programs.

The reference Llama (packages/@affon/models/src/llama/model.ts:64-87) gives
each block seven projections: query, key, value and attentionOutput around
attention, and gate, up and down in the feed-forward
``down(mul(silu(gate(h)), up(h)))``. It stores them dense as ``[in, out]``
matrices for ``matmul``. Quantized checkpoints keep the Hugging Face
``[out, in]`` orientation (packages/@affon/huggingface/src/adapters/llama.ts:27-33),
which is exactly quantized_matmul's packed ``[N, K/P]`` row layout, so here each
projection is one quantized_matmul over ``[out, in]`` packed weights.

Each part of the block is a Program whose weights are arguments:
* ``attention_program``: normalized ``[M, width]`` -> (query, key, value), with
  each projection's output bias when the checkpoint has one
  (``add(quantized_matmul(..), bias)``, lowered into the kernel's epilogue);
* ``output_program``: attention ``[M, width]`` -> attentionOutput;
* ``feed_forward_program``: normalized ``[M, width]`` ->
  ``down(mul(silu(gate), up))``, whose gate/up pair lowers to one fused step
  (one launch at M = 1).

``QuantizedDecoderBlock.step`` runs a whole block over drafted tokens: its
norms (model.ts:64-87 has one before attention and one before the
feed-forward), the rotation with the heads' norms, the append to a paged cache
and the attention, over shared prefixes too, are evaluated ops (cache.py,
``residual_norm``) between those Programs.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Mapping

from . import checkpoint as ckpt
from .cache import (DraftBatch, PagedCache, RotaryAxes, attention_weights, cache_append, shared_attention,
                    tree_attention)
from .core import Program, Session, Tensor, TensorSpec, program
from .ops import add, mul, quantized_matmul, residual_norm, silu

# (block field of LlamaWeights, Hugging Face module, input side, output side)
PROJECTIONS = (
    ("query", "self_attn.q_proj", "width", "width"),
    ("key", "self_attn.k_proj", "width", "kv_width"),
    ("value", "self_attn.v_proj", "width", "kv_width"),
    ("attentionOutput", "self_attn.o_proj", "width", "width"),
    ("gate", "mlp.gate_proj", "width", "inner_width"),
    ("up", "mlp.up_proj", "width", "inner_width"),
    ("down", "mlp.down_proj", "inner_width", "width"),
)

# (norm of a block, Hugging Face module of its weight)
NORMS = {"attentionNorm": "input_layernorm", "feedForwardNorm": "post_attention_layernorm"}
# (norm of a block's query or key heads, Hugging Face module of its weight)
HEAD_NORMS = {"queryNorm": "self_attn.q_norm", "keyNorm": "self_attn.k_norm"}


@dataclass(frozen=True)
class DecoderShape:
    """The dimensions create_llama checks (model.ts:17-20)."""
    width: int
    inner_width: int
    heads: int
    kv_heads: int

    def __post_init__(self):
        dims = (self.width, self.inner_width, self.heads, self.kv_heads)
        if any(not isinstance(d, int) or isinstance(d, bool) or d <= 0 for d in dims):
            raise TypeError("Invalid Llama dimensions, RoPE or normalization")
        if self.width % self.heads or self.heads % self.kv_heads or (self.width // self.heads) % 2:
            raise TypeError("Invalid Llama dimensions, RoPE or normalization")

    @property
    def kv_width(self) -> int:
        return self.kv_heads * (self.width // self.heads)

    def features(self, name: str) -> tuple[int, int]:
        """(out, in) of a projection."""
        for field, _, side_in, side_out in PROJECTIONS:
            if field == name:
                return getattr(self, side_out), getattr(self, side_in)
        raise KeyError(name)


class QuantizedDecoderBlock:
    """The seven quantized projections of one block, with optional output
    biases, and the Programs that run them."""

    def __init__(self, shape: DecoderShape, layers: Mapping[str, ckpt.QuantizedLinear],
                 output_biases: Mapping[str, Tensor] | None = None, norms: Mapping[str, Tensor] | None = None,
                 head_norms: Mapping[str, Tensor] | None = None):
        output_biases, norms, head_norms = dict(output_biases or {}), dict(norms or {}), dict(head_norms or {})
        names = [p[0] for p in PROJECTIONS]
        if sorted(layers) != sorted(names):
            raise TypeError(f"a decoder block needs the projections {names}")
        first = layers[names[0]]
        session = first.packed.session
        for name in names:
            layer = layers[name]
            out_features, in_features = shape.features(name)
            if (layer.out_features, layer.in_features) != (out_features, in_features):
                raise TypeError(f"{name} must be [{out_features}, {in_features}] (out, in), got "
                                f"[{layer.out_features}, {layer.in_features}]")
            if (layer.bits, layer.group_size) != (first.bits, first.group_size):
                raise TypeError("every projection of a block must share bits and group_size")
            if layer.packed.session is not session:
                raise TypeError("every projection of a block must belong to the same Session")
        for name, bias in output_biases.items():
            if name not in names:
                raise TypeError(f"unknown projection {name}")
            if name in ("gate", "up"):
                raise TypeError("gate and up output biases are not supported (the SiLU-gated product fuses them)")
            if bias.dtype not in ("f32", "bf16") or bias.shape != (shape.features(name)[0],):
                raise TypeError(f"{name} output bias must be an f32/bf16 [{shape.features(name)[0]}] tensor")
        for name, weight in norms.items():
            if name not in NORMS:
                raise TypeError(f"unknown norm {name}")
            if weight.dtype not in ("f32", "bf16") or weight.shape != (shape.width,):
                raise TypeError(f"{name} must be an f32/bf16 [{shape.width}] tensor")
        for name, weight in head_norms.items():
            if name not in HEAD_NORMS:
                raise TypeError(f"unknown head norm {name}")
            if weight.dtype not in ("f32", "bf16") or weight.shape not in self._head_norm_shapes(shape, name):
                raise TypeError(f"{name} must be an f32/bf16 tensor of one of the shapes "
                                f"{[list(s) for s in self._head_norm_shapes(shape, name)]}")
        self.norms, self.head_norms = norms, head_norms
        self.unread_norms: tuple[str, ...] = ()  # that a checkpoint does not hold as f32/bf16 [width]
        self.shape = shape
        self.layers = dict(layers)
        self.output_biases = output_biases
        self.bits = first.bits
        self.group_size = first.group_size
        self.session: Session = session
        self._programs: dict[tuple[str, int, str], Program] = {}

    @staticmethod
    def _head_norm_shapes(shape: DecoderShape, name: str) -> tuple[tuple[int], tuple[int]]:
        """Of one weight for all heads, or of each head's own."""
        return (shape.width // shape.heads,), (shape.width if name == "queryNorm" else shape.kv_width,)

    # ---- construction from a checkpoint ----

    @classmethod
    def from_checkpoint(cls, session: Session, path: str, index: int, shape: DecoderShape, *, bits: int,
                        group_size: int, prefix: str = "model.layers",
                        head_norms: bool | None = None) -> "QuantizedDecoderBlock":
        """Binds block ``index`` of an MLX-affine checkpoint: ``<prefix>.<index>.
        <module>.weight`` (U32) with ``.scales`` / ``.biases`` per projection,
        and ``<module>.bias`` as the output bias where present. Norms' weights
        are read where they are f32/bf16 ``[width]``; without them the block runs
        its projections and refuses a ``step``. (A block that is made without
        ``norms`` has norms of ones.) Query and key heads are normed where the
        checkpoint holds weights for it, which are read likewise: one
        ``[head_dim]`` for all heads. (``[heads * head_dim]`` may be each head's own
        or a norm's over the whole projection, which the block does not have, so a
        ``step`` is refused.) ``head_norms`` True: both are needed, of all heads or
        of each; False: neither is read."""
        base = f"{prefix}.{index}"
        modules = {field: f"{base}.{module}" for field, module, _, _ in PROJECTIONS}
        bound = ckpt.quantized_linears(session, path, bits=bits, group_size=group_size, prefixes=modules.values())
        header = ckpt.inspect(path)
        bias_names = [m + ".bias" for m in modules.values() if m + ".bias" in header]
        norm_names = {name: f"{base}.{module}.weight" for name, module in NORMS.items() if f"{base}.{module}.weight" in header}
        # A weight that is not there, or of another type or shape, does not keep
        # the projections from being bound; a step, which needs it, then refuses.
        for name in [n for n in norm_names if header[norm_names[n]]["dtype"] not in ("F32", "BF16")
                     or header[norm_names[n]]["shape"] != [shape.width]]:
            del norm_names[name]
        heads = {name: f"{base}.{module}.weight" for name, module in HEAD_NORMS.items()}
        heads = {name: tensor for name, tensor in heads.items() if head_norms or head_norms is None and tensor in header}
        head_names = {name: tensor for name, tensor in heads.items() if tensor in header and
                      header[tensor]["dtype"] in ("F32", "BF16") and
                      tuple(header[tensor]["shape"]) in cls._head_norm_shapes(shape, name)[:2 if head_norms else 1]}
        wanted = bias_names + list(norm_names.values()) + list(head_names.values())
        loaded = ckpt.load(session, path, wanted) if wanted else {}
        layers = {field: bound[module] for field, module in modules.items()}
        biases = {field: loaded[module + ".bias"] for field, module in modules.items() if module + ".bias" in loaded}
        block = cls(shape, layers, biases, {name: loaded[module] for name, module in norm_names.items()},
                    {name: loaded[module] for name, module in head_names.items()})
        block.unread_norms = tuple(n for n in NORMS if n not in norm_names) + tuple(n for n in heads if n not in head_names)
        return block

    # ---- Programs ----

    def _weights(self, p, name: str):
        layer = self.layers[name]
        return (p.argument(f"{name}.packed", layer.packed.spec), p.argument(f"{name}.scales", layer.scales.spec),
                p.argument(f"{name}.biases", layer.biases.spec))

    def _project(self, p, name: str, x):
        y = quantized_matmul(x, *self._weights(p, name), bits=self.bits, group_size=self.group_size)
        bias = self.output_biases.get(name)
        if bias is not None:
            y = add(y, p.argument(f"{name}.bias", bias.spec))
        return y

    def _program(self, part: str, rows: int, dtype: str) -> Program:
        key = (part, rows, dtype)
        if key not in self._programs:
            width = self.shape.width
            if part == "attention":
                body = lambda p: self._attention_body(p, rows, dtype)
            elif part == "output":
                body = lambda p: self._project(p, "attentionOutput", p.argument("attention",
                                                                                 TensorSpec(dtype, (rows, width))))
            else:
                body = lambda p: self._feed_forward_body(p, rows, dtype)
            self._programs[key] = program(f"quantized_decoder_{part}", body)
        return self._programs[key]

    def _attention_body(self, p, rows: int, dtype: str):
        h = p.argument("normalized", TensorSpec(dtype, (rows, self.shape.width)))
        return [self._project(p, name, h) for name in ("query", "key", "value")]

    def _feed_forward_body(self, p, rows: int, dtype: str):
        h = p.argument("normalized", TensorSpec(dtype, (rows, self.shape.width)))
        gated = mul(silu(self._project(p, "gate", h)), self._project(p, "up", h))
        return self._project(p, "down", gated)

    def attention_program(self, rows: int, dtype: str = "bf16") -> Program:
        return self._program("attention", rows, dtype)

    def output_program(self, rows: int, dtype: str = "bf16") -> Program:
        return self._program("output", rows, dtype)

    def feed_forward_program(self, rows: int, dtype: str = "bf16") -> Program:
        return self._program("feed_forward", rows, dtype)

    def weight_arguments(self) -> dict[str, Tensor]:
        args: dict[str, Tensor] = {}
        for name, layer in self.layers.items():
            args[f"{name}.packed"], args[f"{name}.scales"], args[f"{name}.biases"] = (layer.packed, layer.scales,
                                                                                   layer.biases)
        for name, bias in self.output_biases.items():
            args[f"{name}.bias"] = bias
        return args

    # ---- running ----

    def _run(self, source: Program, inputs: Mapping[str, Tensor], **options):
        # run() reads the arguments its Program names.
        return self.session.compile(source, **options).run({**self.weight_arguments(), **inputs})

    def attention(self, normalized: Tensor, **options) -> list[Tensor]:
        """(query, key, value) of normalized activations [M, width]."""
        return self._run(self.attention_program(normalized.shape[0], normalized.dtype), {"normalized": normalized},
                         **options)

    def attention_output(self, attention: Tensor, **options) -> Tensor:
        return self._run(self.output_program(attention.shape[0], attention.dtype), {"attention": attention},
                         **options)

    def feed_forward(self, normalized: Tensor, **options) -> Tensor:
        """down(silu(gate(h)) * up(h)) of normalized activations [M, width]."""
        return self._run(self.feed_forward_program(normalized.shape[0], normalized.dtype), {"normalized": normalized},
                         **options)

    def step(self, stream: Tensor, update: Tensor | None, cache: PagedCache, batch: DraftBatch, rotary: Tensor, *,
             positions: Tensor | None = None, mask: Tensor | None = None, layer: int = 0, epsilon: float = 1e-5,
             scale: float | None = None, interleaved: bool = False, axes: RotaryAxes | None = None,
             shared: Tensor | None = None, weights: Tensor | None = None, **options) -> tuple[Tensor, Tensor]:
        """The block over a batch's drafted tokens (row b*T + i of ``stream``
        [B*T, width]: token i of sequence b), whose keys and values it appends to
        ``layer`` of the cache. ``update`` is what the block before still adds to
        the stream (None: nothing), and the result (stream, update) what the next
        one takes: every residual add is part of the norm that follows it. After
        the last block, ``residual_norm(stream, update, weight=final)`` gives
        the hidden states, and once their tokens are judged ``cache_commit``
        keeps the accepted ones.

        ``positions`` and ``mask`` as cache_append and tree_attention take them (a
        tree's depths and ancestors; None: a chain); ``axes``: of positions with
        several; ``shared``: tokens that groups of sequences share, as
        shared_attention takes them; ``weights``: gathered ones, to which
        attention_weights adds the rows'. ``options``: the projections' compile
        options."""
        if self.unread_norms:
            shape = f"[{self.shape.width}] " if set(self.unread_norms) <= set(NORMS) else ""
            wider = "" if shape else f" (heads: [{self.shape.width // self.shape.heads}], or with head_norms=True each head's own)"
            raise TypeError(f"the checkpoint holds no f32/bf16 {shape}tensor for {', '.join(self.unread_norms)}{wider}")
        stream, normalized = residual_norm(stream, update, weight=self.norms.get("attentionNorm"), epsilon=epsilon,
                                           dtype=cache.dtype)
        query, key, value = self.attention(normalized, **options)
        rotated = cache_append(cache, batch, query, key, value, positions, rotary, layer=layer,
                               interleaved=interleaved, query_norm=self.head_norms.get("queryNorm"),
                               key_norm=self.head_norms.get("keyNorm"), epsilon=epsilon, axes=axes)
        if shared is None:
            attended = tree_attention(cache, batch, rotated, mask, layer=layer, scale=scale)
        else:
            attended = shared_attention(cache, batch, rotated, shared, mask, layer=layer, scale=scale)
        if weights is not None:
            attention_weights(cache, batch, rotated, weights, mask, layer=layer, scale=scale)
        stream, normalized = residual_norm(stream, self.attention_output(attended, **options),
                                           weight=self.norms.get("feedForwardNorm"), epsilon=epsilon,
                                           dtype=cache.dtype)
        return stream, self.feed_forward(normalized, **options)
