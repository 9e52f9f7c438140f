"""Adapters, beams and states on the CPU: what the entry points refuse before any launch, and their plain forms."""

from __future__ import annotations

import numpy as np
import pytest

from nanocompile_b200 import runtime, serving
from tests import requests_ref as ref
from tests.test_serving import Fake

BATCH, LAYOUT = serving.LoraBatch(5, 5, 4), serving.LoraLayout(64, (32, 16), 8)


def project(**change):
    given = {"out": Fake((5, 48), np.float32, address=8192), "x": Fake((5, 64), np.float32), "a": Fake((4, 16, 64), np.float16),
             "b": Fake((4, 48, 8), np.float16), "plan": Fake((4096,), np.uint8), "layout": LAYOUT, "batch": BATCH, **change}
    serving.lora_project(given.pop("layout"), given.pop("batch"), given.pop("out"), given.pop("x"), given.pop("a"), given.pop("b"),
                         given.pop("plan"), **given)


@pytest.mark.parametrize("change,what", [
    (dict(out=Fake((5, 47), np.float32)), "out: .*expected 5 contiguous rows of 48"), (dict(x=Fake((4, 64), np.float32)), "x: "),
    (dict(x=Fake((5, 64), np.float16)), "different types"), (dict(base=Fake((5, 48), np.float16)), "different types"),
    (dict(base=Fake((5, 49), np.float32)), "base: "), (dict(x=Fake((5, 64), np.int32)), "element type"),
    (dict(x=Fake((5, 64), np.float32, strides=(64, 2))), "contiguous rows"), (dict(x=Fake((5, 64), np.float32, strides=(32, 1))), "overlap"),
    (dict(out=Fake((5, 48), np.float32, strides=(40, 1))), "overlap"), (dict(a=Fake((4, 16, 64), np.float32)), "float16 or bfloat16"),
    (dict(a=Fake((4, 16, 72), np.float16)), "a: "), (dict(b=Fake((4, 48, 16), np.float16)), "b: "), (dict(b=Fake((3, 48, 8), np.float16)), "b: "),
    (dict(a=Fake((4, 16, 64), np.float16, address=4104)), "16-byte boundary"), (dict(plan=Fake((64,), np.uint8)), "plan of 64 bytes"),
    (dict(plan=Fake((4096,), np.uint8, address=4100)), "16-byte boundary"), (dict(plan=Fake((64, 64), np.uint8)), "scratch"),
    (dict(ranks=Fake((3,), np.int32)), "ranks"), (dict(scales=Fake((4,), np.float16)), "scales"),
    (dict(out=Fake((5, 48), np.float32, address=0)), "null output"), (dict(x=Fake((5, 64), np.float32, address=4098)), "misaligned"),
    (dict(x=Fake((5, 64), np.float32, address=8192)), "the outputs are the inputs"),
    (dict(base=Fake((5, 48), np.float32, address=8192, strides=(50, 1))), "in place of base"),
    (dict(layout=serving.LoraLayout(2 ** 23 + 8, (32, 16), 8), x=Fake((5, 2 ** 23 + 8), np.float32), a=Fake((4, 16, 2 ** 23 + 8), np.float16)), "8388608 at most"),
    (dict(layout=serving.LoraLayout(64, (32, 2 ** 23), 8), out=Fake((5, 2 ** 23 + 32), np.float32, address=8192), b=Fake((4, 2 ** 23 + 32, 8), np.float16)),
     "8388608 outputs after 32"),
])
def test_projections_refuse(change, what):
    with pytest.raises(runtime.InterpreterError, match=what):
        project(**change)


@pytest.mark.parametrize("sizes", [(60, (8,), 8), (64, (), 8), (64, (8, 0), 8), (64, (8,), 12), (64, (8,), 136), (64, (8,), 0), (0, (8,), 8),
                                   (64, (1,) * 9, 8)])
def test_adapter_layouts_that_do_not_exist(sizes):
    with pytest.raises(runtime.InterpreterError):
        serving.LoraLayout(*sizes)


@pytest.mark.parametrize("sizes", [(-1, 1, 1), (1, 8193, 1), (1, 1, 0), (1, -1, 1)])
def test_batches_that_do_not_exist(sizes):
    with pytest.raises(runtime.InterpreterError):
        serving.LoraBatch(*sizes)


@pytest.mark.parametrize("change,what", [
    (dict(plan=Fake((32,), np.uint8)), "plan of 32 bytes"), (dict(adapters=Fake((4,), np.int32)), "adapters"), (dict(adapters=Fake((5,), np.int64)), "adapters"),
    (dict(row_start=Fake((5,), np.int32)), "row_start"), (dict(batch=serving.LoraBatch(6, 5, 4)), "need row_start"),
    (dict(error=Fake((1,), np.int32)), "error"), (dict(adapters=Fake((5,), np.int32, address=0)), "null adapters"),
    (dict(batch=serving.LoraBatch(6, 0, 4), adapters=Fake((0,), np.int32)), "of no sequence"),
    (dict(error=Fake((1,), np.uint64, address=4100)), "8-byte boundary")])
def test_plans_refuse(change, what):
    given = {"batch": BATCH, "plan": Fake((4096,), np.uint8), "adapters": Fake((5,), np.int32), **change}
    with pytest.raises(runtime.InterpreterError, match=what):
        serving.lora_plan(given.pop("batch"), given.pop("plan"), given.pop("adapters"), **given)


def test_plan_bytes_hold_every_item_and_row():
    for rows, seqs, slots in ((1, 1, 1), (64, 64, 8), (8192, 8, 5), (8192, 8192, 10000), (0, 0, 1)):
        groups = min(rows, seqs, slots + 1)                              # with a row each; the others fill whole items at best
        assert serving.LoraBatch(rows, seqs, slots).plan_bytes >= 4 * rows + 16 * (groups + (rows - groups) // 128)


@pytest.mark.parametrize("change,what", [
    (dict(parent=Fake((5,), np.int32)), "parent"), (dict(tokens=Fake((6,), np.int32)), "tokens"), (dict(new_scores=Fake((6,), np.float16)), "new_scores"),
    (dict(logits=Fake((6, 50), np.int32)), "element type"), (dict(logits=Fake((6, 50), np.float32, strides=(50, 2))), "contiguous rows"),
    (dict(logits=Fake((6, 50), np.float32, strides=(49, 1))), "overlap"), (dict(beams=4), "whole requests"), (dict(beams=33), "at most 32"), (dict(beams=0), "beams"),
    (dict(end=50), "end token"), (dict(finished=Fake((6,), np.int32)), "without an end token"), (dict(scratch=Fake((64,), np.uint8)), "scratch of 64"),
    (dict(scores=Fake((6,), np.float64)), "scores"), (dict(scores=Fake((6,), np.float32, address=12288)), "are the old ones"),
    (dict(finished=Fake((6,), np.int32), new_finished=Fake((6,), np.int32), end=1), "are the old ones"), (dict(norms=Fake((5,), np.float32)), "norms"),
    (dict(logits=Fake((6, 50), np.float32, address=4098)), "misaligned"), (dict(scratch=Fake((1 << 20,), np.uint8, address=4104)), "scratch"),
    (dict(logits=Fake((6, 0), np.float32)), "0 logits"), (dict(logits=Fake((6, 2 ** 31), np.float32)), "too large for 3 beams")])
def test_selections_refuse(change, what):
    given = {"parent": Fake((6,), np.int32), "tokens": Fake((6,), np.int64), "new_scores": Fake((6,), np.float32, address=12288),
             "logits": Fake((6, 50), np.float32), "scores": Fake((6,), np.float32), "scratch": Fake((1 << 20,), np.uint8), "beams": 3, **change}
    with pytest.raises(runtime.InterpreterError, match=what):
        serving.beam_select(given.pop("parent"), given.pop("tokens"), given.pop("new_scores"), given.pop("logits"), given.pop("scores"),
                            given.pop("scratch"), **given)


@pytest.mark.parametrize("beams", [1, 2, 3, 4, 5, 8, 16, 31, 32])
def test_a_beam_scratch_grows_with_every_size(beams):
    """So that one for some rows, vocabulary and beams serves the calls of fewer of any of them."""
    vocabularies = sorted({*range(1, 300000, 997), 54000, 62000, 66000, 108000, 132000, 234000, 264000})
    for rows in (1, beams, 40 * beams):
        sizes = [serving.beam_select_scratch_bytes(rows, v, beams) for v in vocabularies]
        assert sizes == sorted(sizes)
        assert all(serving.beam_select_scratch_bytes(rows + 1, v, beams) >= s and serving.beam_select_scratch_bytes(rows, v, max(1, beams - 1)) <= s
                   for v, s in zip(vocabularies, sizes))


def test_a_beam_scratch_covers_every_smaller_call():
    sizes = [serving.beam_select_scratch_bytes(r, v, k) for r, v, k in ((1, 100, 1), (1, 151936, 1), (64, 151936, 4), (256, 151936, 8), (4096, 151936, 32))]
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("change,what", [
    (dict(old=Fake((3, 2, 8, 5), np.float32)), "old"), (dict(old=Fake((3, 2, 8, 4), np.float16)), "old"), (dict(parent=Fake((2,), np.int32)), "parent"),
    (dict(old=Fake((3, 2, 8, 4), np.float32, address=8192)), "are the old ones"), (dict(new=Fake((3, 2, 8, 4), np.float32, strides=(64, 33, 4, 1))), "strides"),
    (dict(new=Fake((3, 2, 8, 4), np.float32, strides=(60, 32, 4, 1))), "overlap"), (dict(new=Fake((3, 8, 4), np.float32)), "expected"),
    (dict(new=Fake((3, 2, 8, 4), np.float64)), "expected"), (dict(new_lengths=Fake((3,), np.int32)), "without lengths"),
    (dict(append=Fake((3, 2, 4), np.float32)), "without lengths"), (dict(lengths=Fake((3,), np.int32), append=Fake((3, 4), np.float32)), "append"),
    (dict(lengths=Fake((3,), np.int32), grow=Fake((3,), np.int32)), "grow without"),
    (dict(lengths=Fake((3,), np.int32), new_lengths=Fake((3,), np.int32)), "are the old ones"),
    (dict(new=Fake((2 ** 30, 2 ** 30, 64, 2 ** 16), np.uint8, address=8192, strides=(2 ** 52, 2 ** 22, 2 ** 16, 1)), parent=Fake((2 ** 30,), np.int32),
          old=Fake((2 ** 30, 2 ** 30, 64, 2 ** 16), np.uint8, strides=(2 ** 52, 2 ** 22, 2 ** 16, 1))), "in one call")])
def test_reorders_refuse(change, what):
    given = {"new": Fake((3, 2, 8, 4), np.float32, address=8192), "old": Fake((3, 2, 8, 4), np.float32), "parent": Fake((3,), np.int32), **change}
    with pytest.raises(runtime.InterpreterError, match=what):
        serving.beam_reorder(given.pop("new"), given.pop("old"), given.pop("parent"), **given)


def test_the_plain_forms_agree_with_a_definition_of_their_own():
    rng = np.random.default_rng(0)
    x, a, b = rng.standard_normal((3, 8)), rng.standard_normal((2, 16, 8)), rng.standard_normal((2, 5, 8))
    out, _ = ref.lora(x, a, b, (3, 2), 8, [1, -1, 0], [0, 1, 2, 3])
    assert np.allclose(out[0, 4], sum(b[1, 4, j] * (a[1, 8 + j] @ x[0]) for j in range(8))) and (out[1] == 0).all()
    found = ref.beams(np.log(np.array([[0.5, 0.3, 0.2], [0.9, 0.05, 0.05]])), [0.0, -0.1], 2)[0]
    assert [(c[1], c[2]) for c in found[:2]] == [(1, 0), (0, 0)] and np.isclose(found[0][3], np.log(0.9) - 0.1)
