"""The serving operators on the CPU: the layout's arithmetic, and what the entry points refuse before any launch."""

from __future__ import annotations

import numpy as np
import pytest

from nanocompile_b200 import runtime, serving
from tests import serving_ref as ref


class Fake:
    """An array that exists on no device: its address is only looked at."""

    def __init__(self, shape, dtype, address: int = 4096, strides=None):
        self.shape, self.dtype, self.address = tuple(shape), np.dtype(dtype), address
        self.strides = strides or tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))
        self.dense = strides is None

    def data_ptr(self):
        return self.address

    def stride(self):
        return self.strides

    def is_contiguous(self):
        return self.dense


def cache(layout, seqs=2, width=3, pages=5):
    return (Fake((pages, layout.page_bytes), np.uint8), Fake((seqs, width), np.int32), Fake((seqs,), np.int32))


def attend(layout, rows=2, *, q=None, out=None, scratch=None, table=None, pool=None, lengths=None, **options):
    p, t, n = cache(layout)
    line = layout.heads * layout.head_dim
    serving.kv4_attention(layout, out or Fake((rows, line), np.float32), q or Fake((rows, line), np.float32), pool or p,
                          table or t, lengths or n, scratch or Fake((1 << 20,), np.uint8),
                          **{"max_length": 100, **options})


LAYOUT = serving.KV4Layout(14, 2, 64, 64)


@pytest.mark.parametrize("options,what", [
    (dict(q=Fake((2, 895), np.float32)), "expected rows of 14"),
    (dict(q=Fake((2, 896), np.int32)), "element type"),
    (dict(q=Fake((2, 896), np.float16)), "different types"),
    (dict(q=Fake((2, 896), np.float32, strides=(896, 2))), "expected rows of 14"),
    (dict(out=Fake((3, 896), np.float32)), "3 rows, expected 2"),
    (dict(table=Fake((2, 3), np.int64)), "table"),
    (dict(table=Fake((6,), np.int32)), "table"),
    (dict(lengths=Fake((3,), np.int32)), "lengths"),
    (dict(pool=Fake((5, 10241), np.uint8)), "pool"),
    (dict(layer=1), "layer 1 of 1"),
    (dict(row_start=Fake((2,), np.int32)), "row_start"),
    (dict(max_rows=2), "at most 2 rows"),
    (dict(max_length=-1), "positions of a sequence"),
    (dict(scale=0.0), "score scale"),
    (dict(scale=float("nan")), "score scale"),
    (dict(rope=(Fake((9, 32), np.float32), Fake((9, 31), np.float32))), "sin"),
    (dict(lse=Fake((2, 13), np.float32)), "lse"),
    (dict(pool=Fake((5, LAYOUT.page_bytes), np.uint8, address=4100)), "16-byte boundary"),
    (dict(max_length=100000, scratch=Fake((64,), np.uint8)), "scratch of 64 bytes"),
    (dict(q=Fake((2, 896), np.float32, strides=(800, 1))), "overlap"),
    (dict(q=Fake((2, 896), np.float32, address=0)), "null output or queries"),
])
def test_attention_refuses(options, what):
    with pytest.raises(runtime.InterpreterError, match=what):
        attend(LAYOUT, **options)


def test_a_row_for_each_sequence_needs_no_row_start_and_other_rows_do():
    with pytest.raises(runtime.InterpreterError, match="need row_start"):
        attend(LAYOUT, rows=3)


@pytest.mark.parametrize("sizes,what", [((14, 4, 64), "evenly"), ((0, 1, 64), "evenly"), ((2, 1, 48), "32, 64, 96 and 128"),
                                        ((2, 1, 256), "32, 64, 96 and 128"), ((2, 1, 64, 24), "multiple of 16"),
                                        ((2, 1, 64, 0), "multiple of 16"), ((2, 1, 64, 2048), "1024"), ((2, 1, 64, 64, 0), "evenly")])
def test_layouts_that_do_not_exist(sizes, what):
    with pytest.raises(runtime.InterpreterError, match=what):
        attend(serving.KV4Layout(*sizes))


@pytest.mark.parametrize("change,what", [
    (dict(keys=Fake((2, 127), np.float32)), "keys"), (dict(values=Fake((3, 128), np.float32)), "values"),
    (dict(values=Fake((2, 128), np.float16)), "different types"), (dict(keys=Fake((2, 128), np.float32, address=0)), "null keys"),
    (dict(values=Fake((2, 128), np.float32, strides=(64, 1))), "overlap")])
def test_append_refuses(change, what):
    pool, table, lengths = cache(LAYOUT)
    given = {"keys": Fake((2, 128), np.float32), "values": Fake((2, 128), np.float32), **change}
    with pytest.raises(runtime.InterpreterError, match=what):
        serving.kv4_append(LAYOUT, pool, given["keys"], given["values"], table, lengths)


def test_read_refuses_other_types_and_strides():
    pool, table, lengths = cache(LAYOUT)
    for keys in (Fake((2, 128), np.float16), Fake((2, 128), np.float32, strides=(256, 1))):
        with pytest.raises(runtime.InterpreterError, match="contiguous float32"):
            serving.kv4_read(LAYOUT, keys, keys, pool, table, lengths)


@pytest.mark.parametrize("change,what", [
    (dict(new_table=Fake((2, 4), np.int32)), "new_table"), (dict(new_lengths=Fake((2,), np.int64)), "new_lengths"),
    (dict(status=Fake((3,), np.int64)), "status"), (dict(scratch=Fake((16,), np.uint8)), "scratch of 16 bytes"),
    (dict(pool=Fake((5, 40), np.uint8)), "multiple of 16"), (dict(parent=Fake((3,), np.int32)), "parent"),
    (dict(grow=Fake((2,), np.float32)), "grow"), (dict(new_table=Fake((2, 3), np.int32)), "the new table is the old one"),
    (dict(new_lengths=Fake((2,), np.int32, address=8192)), "the new lengths")])
def test_page_updates_refuse(change, what):
    given = {"new_table": Fake((2, 3), np.int32, address=12288), "new_lengths": Fake((2,), np.int32),
             "table": Fake((2, 3), np.int32), "lengths": Fake((2,), np.int32, address=8192), "pool": Fake((5, 64), np.uint8),
             "status": Fake((4,), np.int64), "scratch": Fake((4096,), np.uint8), "page_size": 16, **change}
    with pytest.raises(runtime.InterpreterError, match=what):
        serving.kv_pages_update(**given)


@pytest.mark.parametrize("change,what", [
    (dict(logits=Fake((2, 50), np.float32, strides=(50, 2))), "contiguous rows"), (dict(logits=Fake((2, 50), np.int64)), "element type"),
    (dict(logits=Fake((2, 50), np.float32, strides=(40, 1))), "overlap"), (dict(targets=Fake((2, 1), np.int32)), "targets"),
    (dict(targets=Fake((3, 1), np.int64)), "targets"), (dict(out=Fake((2, 2), np.float32)), "out"), (dict(top=Fake((2, 33), np.int64), top_logprobs=Fake((2, 33), np.float32)), "33 alternatives"),
    (dict(logits=Fake((2, 4), np.float32)), "no more than the vocabulary"), (dict(entropy=Fake((3,), np.float32)), "entropy"),
    (dict(logits=Fake((2, 100000), np.float32), scratch=Fake((8,), np.uint8)), "scratch of 8 bytes")])
def test_log_probabilities_refuse(change, what):
    given = {"logits": Fake((2, 50), np.float32), "targets": Fake((2, 1), np.int64), "out": Fake((2, 1), np.float32),
             "entropy": Fake((2,), np.float32), "top": Fake((2, 5), np.int64), "top_logprobs": Fake((2, 5), np.float32),
             "scratch": Fake((1 << 22,), np.uint8), **change}
    with pytest.raises(runtime.InterpreterError, match=what):
        serving.token_logprobs(**given)


def test_nothing_to_do_needs_no_device():
    pool, table, lengths = cache(LAYOUT, seqs=0)
    empty = Fake((0, 128), np.float32)
    serving.kv4_append(LAYOUT, pool, empty, empty, table, lengths)
    serving.kv4_read(LAYOUT, empty, empty, pool, table, lengths)
    serving.kv4_attention(LAYOUT, Fake((0, 896), np.float32), Fake((0, 896), np.float32), pool, table, lengths,
                          Fake((256,), np.uint8), max_length=0)
    serving.token_logprobs(Fake((0, 50), np.float32), Fake((0, 1), np.int64), Fake((0, 1), np.float32))
    serving.kv_pages_update(Fake((0, 3), np.int32), Fake((0,), np.int32), Fake((0, 3), np.int32), Fake((0,), np.int32),
                            Fake((5, 64), np.uint8), Fake((4,), np.int64), Fake((4096,), np.uint8), page_size=16)


def test_layout_bytes_are_five_bits_a_value():
    layout = serving.KV4Layout(14, 2, 64, 64, layers=24)
    assert layout.page_bytes * 8 == 24 * 2 * 2 * 64 * 64 * 5
    assert layout.pages_for(0) == 0 and layout.pages_for(64) == 1 and layout.pages_for(65) == 2


@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_reference_cache_reads_what_it_wrote_and_covers_its_bytes(d):
    """The tests' own restatement of the layout: every nibble and parameter has one place, and all bytes are used."""
    rng = np.random.default_rng(d)
    pool = ref.Pool(2, 3, d, 32, fill=0)
    x = rng.standard_normal((2, 40, 3, d)).astype(np.float32)
    table = np.array([[1, 0]])
    pool.append(x[0], x[1], table, [40], [0, 40])
    keys, values = pool.history(table[0], 40)
    for got, given in ((keys, x[0]), (values, x[1])):
        assert np.array_equal(got, ref.stands_for(*ref.quantise(given)))
    full = ref.Pool(1, 1, d, 16, fill=0)
    for t in range(16):
        for which in range(2):
            full.put(0, 0, 0, t, which, np.full((d // 32, 32), 15), np.full(d // 32, np.float16(np.nan)), np.full(d // 32, np.float16(np.nan)))
    assert (full.bytes != 0).sum() >= 18 * d           # all code bytes; a NaN's low byte may be 0


def test_quantisation_error_is_half_a_step():
    x = np.random.default_rng(0).standard_normal((100, 128)).astype(np.float32) * 3 + 5
    code, scale, zero = ref.quantise(x)
    step = np.repeat(scale.astype(np.float32), 32, -1).reshape(x.shape)
    # Half a step, and what the ends lose to parameters rounded to f16: half a unit of the zero, 15 of the scale's.
    slack = np.abs(x).max() * 2.0 ** -11 + 15 * step * 2.0 ** -11
    assert (np.abs(ref.stands_for(code, scale, zero) - x) <= step / 2 + slack).all()


@pytest.mark.parametrize("heads,kv,d", [(14, 2, 64), (32, 8, 128), (12, 4, 96), (4, 2, 32)])
def test_attention_scratch_covers_smaller_calls(heads, kv, d):
    """Sequences leave a batch, steps have fewer rows, histories are shorter: the size for the largest call is enough."""
    layout = serving.KV4Layout(heads, kv, d)

    def size(seqs, length, rows):
        return serving.kv4_attention_scratch_bytes(layout, seqs * rows, seqs, length, rows)

    assert size(32, 2048, 1) <= size(64, 2048, 1)
    seqs, rows, lengths = [1, 2, 3, 5, 8, 13, 24, 32, 48, 64, 100, 256, 700], [1, 2, 3, 5, 16, 33, 64, 200, 512, 1000], [1, 16, 64, 100, 257, 700, 2048, 6001, 32768]
    for sizes in ((seqs, [1], lengths), (seqs[:7], rows, lengths)):
        for a in range(1, len(sizes[0])):
            for r in range(len(sizes[1])):
                for n in range(1, len(sizes[2])):
                    here = size(sizes[0][a], sizes[2][n], sizes[1][r])
                    assert size(sizes[0][a - 1], sizes[2][n], sizes[1][r]) <= here
                    assert size(sizes[0][a], sizes[2][n - 1], sizes[1][r]) <= here
                    assert r == 0 or size(sizes[0][a], sizes[2][n], sizes[1][r - 1]) <= here


@pytest.mark.parametrize("vocab", [300, 32000, 50257, 128256, 151936, 2000000])
def test_log_probability_scratch_covers_fewer_rows(vocab):
    rows = [1, 2, 3, 5, 6, 8, 12, 16, 24, 32, 50, 64, 100, 128, 200, 253, 256, 300, 507, 512, 592, 1000, 4095, 4096, 4097, 9000]
    for k in (0, 1, 20, 32):
        sizes = [serving.token_logprobs_scratch_bytes(n, vocab, k) for n in rows]
        assert sizes == sorted(sizes)
        assert k == 0 or all(serving.token_logprobs_scratch_bytes(n, vocab, k - 1) <= size for n, size in zip(rows, sizes))


ROWS = Fake((2, 128), np.float32)


@pytest.mark.parametrize("error,what", [(Fake((1,), np.int32), "error: int32"), (Fake((2,), np.float32), "error: float32"), (Fake((0,), np.uint64), "error: uint64"),
                                        (Fake((1,), np.uint64, address=4100), "8-byte boundary"), (Fake((1,), np.int64, address=4092), "8-byte boundary")])
def test_an_error_word_has_64_bits(error, what):
    pool, table, lengths = cache(LAYOUT)
    for call in (lambda: attend(LAYOUT, error=error),
                 lambda: serving.kv4_append(LAYOUT, pool, ROWS, ROWS, table, lengths, error=error),
                 lambda: serving.kv4_read(LAYOUT, ROWS, ROWS, pool, table, lengths, error=error),
                 lambda: serving.token_logprobs(Fake((2, 50), np.float32), Fake((2, 1), np.int64), Fake((2, 1), np.float32), error=error)):
        with pytest.raises(runtime.InterpreterError, match=what):
            call()


@pytest.mark.parametrize("scratch", [Fake((1 << 22,), np.uint8, strides=(0,)), Fake((1 << 22, 2), np.uint8), Fake((), np.uint8)])
def test_scratch_is_contiguous_bytes(scratch):
    two = Fake((2, 3), np.int32)
    for call in (lambda: attend(LAYOUT, scratch=scratch),
                 lambda: serving.token_logprobs(Fake((2, 50), np.float32), Fake((2, 1), np.int64), Fake((2, 1), np.float32), scratch=scratch),
                 lambda: serving.kv_pages_update(two, Fake((2,), np.int32), Fake((2, 3), np.int32, address=8192), Fake((2,), np.int32, address=8192),
                                                 Fake((5, 64), np.uint8), Fake((4,), np.int64), scratch, page_size=16),
                 lambda: serving.kv_pages_compact(two, Fake((2, 3), np.int32, address=8192), Fake((2,), np.int32), Fake((5, 64), np.uint8),
                                                  Fake((4,), np.int64), scratch, page_size=16)):
        with pytest.raises(runtime.InterpreterError, match="scratch: uint8"):
            call()


@pytest.mark.parametrize("change", [dict(top=None), dict(top_logprobs=None), dict(out=None)])
def test_outputs_of_log_probabilities_come_in_pairs(change):
    given = {"logits": Fake((2, 50), np.float32), "targets": Fake((2, 1), np.int64), "out": Fake((2, 1), np.float32),
             "top": Fake((2, 5), np.int64), "top_logprobs": Fake((2, 5), np.float32), "scratch": Fake((1 << 22,), np.uint8), **change}
    with pytest.raises(runtime.InterpreterError, match="top with top_logprobs"):
        serving.token_logprobs(**given)


def test_rows_of_no_sequence_are_refused():
    pool, table, lengths = cache(LAYOUT, seqs=0)
    start = Fake((1,), np.int32)
    for call in (lambda: attend(LAYOUT, table=table, lengths=lengths, row_start=start),
                 lambda: serving.kv4_append(LAYOUT, pool, ROWS, ROWS, table, lengths, row_start=start),
                 lambda: serving.kv4_read(LAYOUT, ROWS, ROWS, pool, table, lengths, row_start=start)):
        with pytest.raises(runtime.InterpreterError, match="2 rows of no sequence"):
            call()
