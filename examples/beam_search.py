"""Beam search on the GPU over a paged 4-bit key/value cache: ``python examples/beam_search.py [beams] [tokens] [requests]``.

A small int8 Qwen2-shaped decoder with random weights, run from the library's fused groups; its history is held by the
serving operators (``nanocompile_b200.serving``). One prompt is prefilled into the first sequence and forked into
``beams``; each step appends and attends over the 4-bit cache, takes every beam's best tokens with their log
probabilities, and hands the pages of the beams that go on to their successors. Only token ids, scores and parents
cross to the host.

With several requests (:func:`beam_search_requests`) the beams are chosen on the device too, and each request may have a
low-rank adapter of its own beside the shared projections; the token histories come to the host at the end.
"""

from __future__ import annotations

import ctypes
import sys
from dataclasses import dataclass
from pathlib import Path

import numpy as np

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from nanocompile_b200 import model, quantize, runtime, serving
from nanocompile_b200.serving import DeviceArray


@dataclass
class Beam:
    tokens: list[int]
    score: float                       # the sum of its tokens' log probabilities


class Adapters:
    """Low-rank adapters of a model's q, k, v, o and down projections: ``slots`` of them, with ranks of their own. Gate and up have none,
    as their fused product leaves neither's output to add to."""

    NAMES = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.down_proj")

    def __init__(self, shape: model.ModelShape, slots: int, rank: int, seed: int = 0):
        rng = np.random.default_rng(seed)
        self.slots = slots
        self.ranks = DeviceArray.of(np.array([max(1, rank >> s % 3) for s in range(slots)], np.int32))
        self.scales = DeviceArray.of(np.full(slots, 2.0, np.float32))
        inputs = {"self_attn.o_proj": shape.q_rows, "mlp.down_proj": shape.inter}
        outputs = {"self_attn.q_proj": shape.q_rows, "self_attn.k_proj": shape.kv_rows, "self_attn.v_proj": shape.kv_rows}
        self.layouts, self.weights = {}, {}
        for name in self.NAMES:
            k, n = inputs.get(name, shape.hidden), outputs.get(name, shape.hidden)
            self.layouts[name] = layout = serving.LoraLayout(k, (n,), rank)
            for layer in range(shape.layers):
                self.weights[layer, name] = [DeviceArray.of((rng.standard_normal(size) * scale).astype(np.float16))
                                             for size, scale in ((layout.a_shape(slots), k ** -0.5), (layout.b_shape(slots), 0.05))]


class Decoder:
    """An int8 decoder over a 4-bit paged cache of ``seqs`` sequences of up to ``length`` positions; ``adapters`` beside its
    projections, one for each sequence (:meth:`use`)."""

    def __init__(self, shape: model.ModelShape, weights: dict[str, np.ndarray], seqs: int, length: int, page_size: int = 16,
                 top: int = 8, adapters: Adapters | None = None):
        self.shape, self.seqs, self.length, self.top = shape, seqs, length, top
        self.lib = runtime.library()
        self.layout = serving.KV4Layout(shape.heads, shape.kv_heads, shape.head_dim, page_size, shape.layers)
        int8 = quantize.int8_projection_weights(weights, shape)
        self.weights = {k: self._packed(v) if k.endswith("@int8") else DeviceArray.of(v) for k, v in int8.items()}
        width = self.layout.pages_for(length)
        pages = seqs * (width + 1)
        self.pool = DeviceArray((pages, self.layout.page_bytes), np.uint8)
        self.tables = [DeviceArray.of(np.full((seqs, width), -1, np.int32)) for _ in range(2)]       # now, and after the next update
        self.lengths = [DeviceArray.zeros((seqs,), np.int32) for _ in range(2)]
        self.status, self.error = DeviceArray.zeros((4,), np.int64), DeviceArray.of(np.array([2**64 - 1], np.uint64))
        self.pages_scratch = DeviceArray.zeros((serving.kv_pages_scratch_bytes(seqs, width, pages),), np.uint8)
        angles = np.arange(length, dtype=np.float32)[:, None] * shape.rope_rates()
        self.rope = DeviceArray.of(np.cos(angles)), DeviceArray.of(np.sin(angles))
        self.rows = 0
        self.adapters, self.adapter_ids = adapters, DeviceArray.of(np.full(seqs, -1, np.int32))

    def use(self, adapters) -> None:
        """The adapter of each sequence from now on (-1: none)."""
        self.adapter_ids.upload(np.asarray(adapters, np.int32))

    def _packed(self, values: np.ndarray) -> DeviceArray:
        out, values = DeviceArray(values.shape, np.uint8), np.ascontiguousarray(values)
        runtime.check(self.lib.nc_pack_int8_weights(out.data_ptr(), values.ctypes.data, values.nbytes))
        return out

    def _group(self, name: str, arrays, sizes) -> None:
        p = (ctypes.c_void_p * len(arrays))(*[a.data_ptr() if a is not None else None for a in arrays])
        runtime.check(getattr(self.lib, name)(p, (ctypes.c_int64 * len(sizes))(*sizes), None))

    def _room(self, rows: int) -> None:
        """The activations of ``rows`` token rows."""
        if rows == self.rows:
            return
        s, f32 = self.shape, np.float32
        self.rows = rows
        wide = max(s.inter, s.hidden, s.q_rows)
        self.x, self.x2, self.normed = (DeviceArray((rows, s.hidden), f32) for _ in range(3))
        self.q, self.ctx = DeviceArray((rows, s.q_rows), f32), DeviceArray((rows, s.q_rows), f32)
        self.k, self.v = (DeviceArray((rows, s.kv_rows), f32) for _ in range(2))
        self.mlp = DeviceArray((rows, s.inter), f32)
        self.xq, self.xs, self.offset = DeviceArray((rows, wide), np.int8), DeviceArray((rows, wide // 32), f32), DeviceArray((rows,), f32)
        self.ids, self.row_start = DeviceArray((rows,), np.int64), DeviceArray((self.seqs + 1,), np.int32)
        self.logits = DeviceArray((rows, s.vocab), f32)
        self.head_scratch = DeviceArray.zeros((self.lib.nc_lm_head_scratch_bytes(rows, s.vocab),), np.uint8)
        self.top_ids, self.top_logprobs = DeviceArray((rows, self.top), np.int64), DeviceArray((rows, self.top), f32)
        self.targets, self.logprobs, self.entropy = DeviceArray((rows, 1), np.int64), DeviceArray((rows, 1), f32), DeviceArray((rows,), f32)
        self.score_scratch = DeviceArray.zeros((serving.token_logprobs_scratch_bytes(rows, s.vocab, self.top),), np.uint8)
        self.attention_scratch = DeviceArray.zeros(
            (serving.kv4_attention_scratch_bytes(self.layout, rows, self.seqs, self.length, rows),), np.uint8)
        if self.adapters:
            self.batch = serving.LoraBatch(rows, self.seqs, self.adapters.slots)
            self.plan = DeviceArray((self.batch.plan_bytes,), np.uint8)

    def _adapt(self, layer: int, name: str, out, x) -> None:
        if self.adapters:
            a, b = self.adapters.weights[layer, name]
            serving.lora_project(self.adapters.layouts[name], self.batch, out, x, a, b, self.plan, base=out, ranks=self.adapters.ranks,
                                 scales=self.adapters.scales)

    def _project(self, out, name: str, n: int, k: int, epilogue: int, operand=None, second=None) -> None:
        w = self.weights
        self._group("nc_matmul_i8_vnni", [out, self.xq, self.xs, self.offset, w[f"{name}@int8"], w[f"{name}@scales"], operand, second],
                    [self.rows, n, k, epilogue])

    def update(self, parent, grow) -> None:
        """Sequences continue ``parent`` (-1: none) with ``grow`` more positions; raises if the pool has too few pages."""
        parent, grow = (v if isinstance(v, DeviceArray) else DeviceArray.of(np.asarray(v, np.int32)) for v in (parent, grow))
        serving.kv_pages_update(self.tables[1], self.lengths[1], self.tables[0], self.lengths[0], self.pool, self.status,
                                self.pages_scratch, page_size=self.layout.page_size, parent=parent, grow=grow)
        missing = int(self.status.numpy()[0])
        if missing:
            raise runtime.InterpreterError(f"the cache lacks {missing} pages")
        self.tables.reverse()
        self.lengths.reverse()

    def step(self, ids, counts, targets=None) -> None:
        """Token rows ``ids`` (on the host or the device), the last ``counts[i]`` positions of each sequence i (already grown by
        :meth:`update`); leaves the rows' logits and top tokens, and the log probabilities of ``targets``, on the device."""
        s, w, at = self.shape, self.weights, (self.tables[0], self.lengths[0])
        self._room(sum(counts))
        rows, eps = self.rows, int(np.array([s.eps], np.float32).view(np.uint32)[0])
        if not isinstance(ids, DeviceArray):
            self.ids.upload(np.asarray(ids, np.int64))
            ids = self.ids
        self.row_start.upload(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        if self.adapters:                                            # the rows of each adapter, for all layers and projections
            serving.lora_plan(self.batch, self.plan, self.adapter_ids, row_start=self.row_start)
        normed = self.normed if self.adapters else None              # the adapters' products take what is not quantised
        self._group("nc_gather_rows", [self.x, ids, w["model.embed_tokens.weight"], self.error], [rows, s.vocab, s.hidden])
        for layer in range(s.layers):
            p = f"model.layers.{layer}"
            self._group("nc_rms_norm_quantize", [normed, self.x, w[f"{p}.input_layernorm.weight"], self.xq, self.xs, self.offset, None],
                        [rows, s.hidden, eps])
            for out, name, n in ((self.q, "q_proj", s.q_rows), (self.k, "k_proj", s.kv_rows), (self.v, "v_proj", s.kv_rows)):
                self._project(out, f"{p}.self_attn.{name}.weight", n, s.hidden, 1, w[f"{p}.self_attn.{name}.bias"])
                self._adapt(layer, f"self_attn.{name}", out, normed)
            serving.kv4_append(self.layout, self.pool, self.k, self.v, *at, row_start=self.row_start, rope=self.rope, layer=layer)
            serving.kv4_attention(self.layout, self.ctx, self.q, self.pool, *at, self.attention_scratch, max_length=self.length,
                                  row_start=self.row_start, max_rows=rows, rope=self.rope, layer=layer)
            self._group("nc_quantize_blocks", [self.xq, self.ctx, self.xs, self.offset, None], [rows, s.q_rows])
            self._project(self.x2, f"{p}.self_attn.o_proj.weight", s.hidden, s.q_rows, 2, self.x)
            self._adapt(layer, "self_attn.o_proj", self.x2, self.ctx)
            self._group("nc_rms_norm_quantize", [None, self.x2, w[f"{p}.post_attention_layernorm.weight"], self.xq, self.xs, self.offset, None],
                        [rows, s.hidden, eps])
            self._project(self.mlp, f"{p}.mlp.gate_proj.weight", s.inter, s.hidden, 3, w[f"{p}.mlp.up_proj.weight@int8"],
                          w[f"{p}.mlp.up_proj.weight@scales"])
            self._group("nc_quantize_blocks", [self.xq, self.mlp, self.xs, self.offset, None], [rows, s.inter])
            self._project(self.x, f"{p}.mlp.down_proj.weight", s.hidden, s.inter, 2, self.x2)
            self._adapt(layer, "mlp.down_proj", self.x, self.mlp)
        self._group("nc_rms_norm_quantize", [self.normed, self.x, w["model.norm.weight"], None, None, None, None], [rows, s.hidden, eps])
        self._group("nc_lm_head_argmax", [self.logits, self.normed, w["model.embed_tokens.weight"], None, self.head_scratch],
                    [rows, s.vocab, s.hidden])
        self.targets.upload(np.zeros((rows, 1), np.int64) if targets is None else np.asarray(targets, np.int64).reshape(rows, 1))
        serving.token_logprobs(self.logits, self.targets, self.logprobs, self.entropy, self.top_ids, self.top_logprobs,
                               scratch=self.score_scratch)


def prefill(decoder: Decoder, prompt, targets=None) -> None:
    """``prompt`` as the first sequence of an otherwise empty cache."""
    none = [-1] * decoder.seqs
    decoder.update(none, [0] * decoder.seqs)
    first = [len(prompt)] + [0] * (decoder.seqs - 1)
    decoder.update(range(decoder.seqs), first)
    decoder.step(prompt, first, targets)


def beam_search(decoder: Decoder, prompt, tokens: int) -> list[Beam]:
    """The best continuations of ``prompt`` by ``tokens`` tokens that a search as wide as the cache finds, best first."""
    n = decoder.seqs
    prefill(decoder, prompt)
    ids, logprobs = decoder.top_ids.numpy()[-1], decoder.top_logprobs.numpy()[-1]
    beams = [Beam([int(t)], float(p)) for t, p in zip(ids[:n], logprobs[:n])]
    parent = [0] * len(beams) + [-1] * (n - len(beams))
    for step in range(tokens - 1):
        decoder.update(parent, [1] * len(beams) + [0] * (n - len(beams)))
        decoder.step([b.tokens[-1] for b in beams], [1] * len(beams) + [0] * (n - len(beams)))
        ids, logprobs = decoder.top_ids.numpy(), decoder.top_logprobs.numpy()
        every = [(b.score + float(logprobs[i, j]), i, int(ids[i, j])) for i, b in enumerate(beams) for j in range(decoder.top)]
        every.sort(key=lambda c: (-c[0], c[1], c[2]))
        parent = [i for _, i, _ in every[:n]] + [-1] * max(0, n - len(every))
        beams = [Beam(beams[i].tokens + [t], score) for score, i, t in every[:n]]
    return beams


def beam_search_requests(decoder: Decoder, prompts, beams: int, tokens: int, adapters=None, end: int = -1) -> list[list[Beam]]:
    """The best continuations of each of several prompts, of up to ``tokens`` tokens or to the token ``end``, best first: request g has
    the cache's sequences ``g * beams ..``, and of a decoder's adapters ``adapters[g]``. The choice, the histories and the
    pages stay on the device."""
    n, groups = decoder.seqs, len(prompts)
    first = [0 if i % beams else len(prompts[i // beams]) - 1 for i in range(n)]
    if adapters is not None:
        decoder.use([adapters[i // beams] for i in range(n)])
    decoder.update([-1] * n, [0] * n)
    decoder.update(range(n), first)
    if any(first):
        decoder.step([t for p in prompts for t in p[:-1]], first)
    # The prompts' last tokens, and from there on the chosen ones: the first beam of each request is the only one to begin with.
    decoder.update(range(n), [int(i % beams == 0) for i in range(n)])
    ids = DeviceArray.of(np.array([prompts[i // beams][-1] for i in range(n)], np.int64))
    scores = [DeviceArray.of(np.where(np.arange(n) % beams == 0, 0, -np.inf).astype(np.float32)), DeviceArray((n,), np.float32)]
    finished = [DeviceArray.zeros((n,), np.int32) for _ in range(2)]
    histories = [DeviceArray.zeros((n, tokens), np.int64) for _ in range(2)]
    lengths = [DeviceArray.zeros((n,), np.int32) for _ in range(2)]
    parent, grow, pages, more = DeviceArray((n,), np.int32), DeviceArray((n,), np.int32), DeviceArray((n,), np.int32), DeviceArray.of(np.ones(n, np.int32))
    scratch = DeviceArray.zeros((serving.beam_select_scratch_bytes(n, decoder.shape.vocab, beams),), np.uint8)
    for step in range(tokens):
        decoder.step(ids, [1] * n)
        serving.beam_select(parent, ids, scores[1], decoder.logits, scores[0], scratch, beams=beams, end=end,
                            finished=finished[0] if end >= 0 else None, new_finished=finished[1], grow=grow, history=pages)
        serving.beam_reorder(histories[1], histories[0], parent, lengths=lengths[0], new_lengths=lengths[1], append=ids, grow=grow)
        for pair in (scores, finished, histories, lengths):
            pair.reverse()
        if step + 1 < tokens:
            decoder.update(pages, more)
    found = zip(histories[0].numpy(), lengths[0].numpy(), scores[0].numpy())
    every = [Beam([int(t) for t in history[:length]], float(score)) for history, length, score in found]
    return [every[g * beams: (g + 1) * beams] for g in range(groups)]


def main(beams: int = 4, tokens: int = 24, requests: int = 1) -> None:
    shape = model.SMALL
    prompt = model.synthetic_prompt(shape.vocab, 37)
    if requests > 1:
        adapters = Adapters(shape, slots=3, rank=16)
        decoder = Decoder(shape, model.synthetic_weights(shape, seed=3, std=0.08), beams * requests, len(prompt) + tokens, adapters=adapters)
        prompts = [prompt[: len(prompt) - g] for g in range(requests)]
        for g, found in enumerate(beam_search_requests(decoder, prompts, beams, tokens, adapters=[g % 4 - 1 for g in range(requests)], end=5)):
            for beam in found:
                print(f"{g}: {beam.score:9.4f}  {' '.join(map(str, beam.tokens))}")
        return
    decoder = Decoder(shape, model.synthetic_weights(shape, seed=3, std=0.08), beams, len(prompt) + tokens)
    for beam in beam_search(decoder, prompt, tokens):
        print(f"{beam.score:9.4f}  {' '.join(map(str, beam.tokens))}")
    _, used, copied, highest = decoder.status.numpy().tolist()
    print(f"{used} pages of {decoder.layout.page_bytes} bytes in use (ids up to {highest - 1}); the last step copied {copied}")


if __name__ == "__main__":
    main(*map(int, sys.argv[1:]))
