"""The serving operators on the GPU against their plain forms in 64 bits (``serving_ref``).

Where a test allows a difference, its bound comes from the roundings that the kernel is allowed:

* Attention of float32 and float16 rows. A score is off by at most 2^-20 of S = max sum_i |q_i k_i| scale (q in 22
  bits, a dozen float32 roundings), so a probability by a factor 1 +- 2^-19 (S + 4), the 4 for its exponential and its own
  22 bits; their weighted mean of values of at most V is then off by at most 2^-18 (S + 4) V.
* bfloat16 rows: q and p round to 11 bits each, 2^-12 relative: 2^-11 (S + 1) V twice, and the same 2^-18 below them.
* The output rounds to its type: half of 2^-23, 2^-10 or 2^-7 of its size.
"""

from __future__ import annotations

import numpy as np
import pytest

from nanocompile_b200 import serving
from nanocompile_b200.serving import DeviceArray, KV4Layout
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]
ALL_ONES = np.uint64(0xFFFFFFFFFFFFFFFF)
ROUNDING = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def attention_bound(dtype, out, size, most):
    bound = 2.0 ** -18 * (size + 4)
    if dtype == "bfloat16":
        bound = bound + 2 * 2.0 ** -11 * (size + 1)
    return bound[..., None] * most + ROUNDING[dtype] * np.abs(out) * 1.001 + 1e-30


def table_of(rng, lengths, page, spare=3, width=None):
    """A page table of pages in any order, and the pool's size."""
    needed = [-(-n // page) for n in lengths]
    count = sum(needed) + spare
    order = rng.permutation(count)
    width = width or max(1, *needed)
    table = np.full((len(lengths), width), -1, np.int32)
    at = 0
    for i, n in enumerate(needed):
        table[i, :n] = order[at: at + n]
        at += n
    return table, count


def starts_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def error_word():
    return DeviceArray.of(np.array([ALL_ONES]))


class Case:
    """A cache with its history made by the plain append, on the device."""

    def __init__(self, rng, lengths, kv, d, page, layers=1, layer=0, fill=0xFF, scale=1.0, width=None):
        self.lengths, self.layer = np.array(lengths, np.int32), layer
        self.table, count = table_of(rng, lengths, page, width=width)
        self.pool = ref.Pool(count, kv, d, page, layers, fill)
        starts = starts_of(lengths)
        keys, values = (rng.standard_normal((2, starts[-1], kv, d)) * scale).astype(np.float32)
        self.pool.append(keys, values, self.table, self.lengths, starts, layer=layer)
        self.histories = [self.pool.history(self.table[i], n, layer) for i, n in enumerate(lengths)]
        self.upload()

    def upload(self):
        self.d_pool, self.d_table = DeviceArray.of(self.pool.bytes), DeviceArray.of(self.table)
        self.d_lengths = DeviceArray.of(self.lengths)

    def attend(self, layout, q, dtype, counts=None, rope=None, scale=None, stride=None, scratch=None, max_length=None, error=None,
               max_rows=None):
        """Output [rows, heads, d] and log-sums of the device's attention."""
        rows, heads, d = q.shape
        counts = [1] * len(self.lengths) if counts is None else counts
        line = heads * d
        host = np.zeros((rows, stride or line), np.float32)
        host[:, :line] = q.reshape(rows, line)
        given = Rows(DeviceArray.of(ref.encode(host, dtype), dtype), line)
        out = DeviceArray.zeros((rows, line), dtype)
        lse = DeviceArray.of(np.full((rows, heads), 7.0, np.float32))
        most = int(self.lengths.max()) if max_length is None else max_length
        most_rows = max(counts) if max_rows is None else max_rows
        if scratch is None:
            scratch = DeviceArray.zeros((serving.kv4_attention_scratch_bytes(layout, rows, len(counts), most, most_rows),), np.uint8)
        single = all(c == 1 for c in counts) and most_rows == 1
        serving.kv4_attention(layout, out, given, self.d_pool, self.d_table, self.d_lengths, scratch, max_length=most,
                              row_start=None if single else DeviceArray.of(starts_of(counts)), max_rows=most_rows,
                              rope=None if rope is None else tuple(DeviceArray.of(t) for t in rope), layer=self.layer,
                              scale=scale, lse=lse, error=error)
        return ref.decode(out.numpy(), dtype).reshape(rows, heads, d), lse.numpy()

    def check(self, layout, q, dtype, counts=None, rope=None, scale=None, **options):
        counts = [1] * len(self.lengths) if counts is None else counts
        q = ref.decode(ref.encode(q, dtype), dtype)
        got, lse = self.attend(layout, q, dtype, counts, rope, scale, **options)
        want, want_lse, size = ref.attention(q, self.histories, self.lengths, starts_of(counts),
                                             np.float32(q.shape[-1] ** -0.5 if scale is None else scale), rope)
        most = max([np.abs(v).max() for _, v in self.histories if v.size] or [0.0])
        off = np.abs(got - want)
        bound = attention_bound(dtype, want, size, most)
        assert (off <= bound).all(), f"off by {(off / bound).max():.2f} of the bound"
        empty = np.isneginf(want_lse)
        assert np.array_equal(np.isneginf(lse), empty) and not got[empty].any()
        slack = (2.0 ** -18 if dtype != "bfloat16" else 2.0 ** -11) * (size + 4)
        a, b = lse[~empty], want_lse[~empty]
        assert (np.abs(a - b) <= slack[~empty] + 2.0 ** -22 * np.abs(b)).all()
        return got, lse


class Rows:
    """The first ``line`` elements of each row of a device array."""

    def __init__(self, array, line):
        self.array, self.shape, self.dtype = array, (array.shape[0], line), array.dtype

    def data_ptr(self):
        return self.array.data_ptr()

    def stride(self):
        return self.array.stride()

    def is_contiguous(self):
        return self.shape[1] == self.array.shape[1]


# -- append and read ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kv,d,page,rotated", [(2, 64, 64, True), (1, 32, 16, False), (3, 96, 48, True), (5, 128, 1024, True)])
def test_append_writes_the_reference_bytes_and_no_others(cuda, dtype, kv, d, page, rotated):
    rng = np.random.default_rng(kv * d)
    counts, before = [3, 0, 17, 1, 5], [0, 9, 14, 2 * page - 1, -3]           # the last: its first rows are before position 0
    lengths = np.array([b + c for b, c in zip(before, counts)], np.int32)
    table, pages = table_of(rng, np.maximum(lengths, 0), page)
    layout = KV4Layout(kv, kv, d, page, layers=2)
    pool = ref.Pool(pages, kv, d, page, 2, fill=0xA5)
    starts = starts_of(counts)
    rows, line = int(starts[-1]), kv * d
    x = ref.encode(rng.standard_normal((rows, 2 * line + 7)).astype(np.float32) * 3, dtype)
    keys, values = (ref.decode(np.ascontiguousarray(v), dtype).reshape(rows, kv, d) for v in (x[:, :line], x[:, line: 2 * line]))
    rope = ref.rope_tables(int(lengths.max()), d) if rotated else None
    d_pool, d_x, error = DeviceArray.of(pool.bytes), DeviceArray.of(x, dtype), error_word()

    class Part(Rows):
        def data_ptr(self):
            return self.array.data_ptr() + line * x.itemsize

    args = (DeviceArray.of(table), DeviceArray.of(lengths))
    d_starts = DeviceArray.of(starts)
    serving.kv4_append(layout, d_pool, Rows(d_x, line), Part(d_x, line), *args, row_start=d_starts, layer=1, error=error,
                       rope=None if rope is None else tuple(DeviceArray.of(t) for t in rope))
    pool.append(keys, values, table, lengths, starts, rope, layer=1)
    assert np.array_equal(d_pool.numpy(), pool.bytes)
    assert error.numpy()[0] == ALL_ONES
    back = [DeviceArray.of(np.full((rows, line), 5, np.float32)) for _ in range(2)]
    serving.kv4_read(layout, *back, d_pool, *args, row_start=d_starts, layer=1)
    for which, got in enumerate(back):
        got = got.numpy().reshape(rows, kv, d)
        for i, n in enumerate(lengths):
            for r in range(starts[i], starts[i + 1]):
                t = n - (starts[i + 1] - r)
                want = np.zeros((kv, d)) if t < 0 else np.stack([pool.get(table[i, t // page], 1, h, t % page, which) for h in range(kv)])
                assert np.array_equal(got[r], want)


@pytest.mark.parametrize("rows_of", ["few", "many"])
@pytest.mark.parametrize("dtype,kv,d,page,rotated,odd", [("float32", 2, 64, 32, True, 0), ("bfloat16", 3, 128, 64, True, 0), ("bfloat16", 1, 96, 16, True, 8),
                                                         ("float16", 2, 32, 16, True, 1), ("float16", 1, 128, 48, False, 3), ("float32", 1, 32, 16, False, 0)])
def test_appends_of_few_and_many_rows_write_the_reference_bytes(cuda, rows_of, dtype, kv, d, page, rotated, odd):
    """Both kernels of the append: ragged sequences, rows before position 0, a missing page, an end of the angles, and blocks
    that f16 parameters hold badly (far from nought, tiny, huge, with infinities)."""
    rng = np.random.default_rng(d + kv)
    counts, before = ([1500, 0, 33, 700], [5, 9, -20, 31]) if rows_of == "many" else ([21, 0, 5, 33, 1], [30, 9, -3, 0, 15])
    lengths = np.array([b + c for b, c in zip(before, counts)], np.int32)
    table, pages = table_of(rng, np.maximum(lengths, 0), page)
    missing = (0, (before[0] + 20) // page)                                       # a page of sequence 0
    layout, pool = KV4Layout(kv, kv, d, page), ref.Pool(pages, kv, d, page, fill=0xA5)
    starts, line = starts_of(counts), kv * d
    rows = int(starts[-1])
    host = rng.standard_normal((rows, 2, line)).astype(np.float32) * 3
    kind = rng.integers(0, 12, rows)
    host[kind == 0] = host[kind == 0] * 1e-3 + 1000
    host[kind == 1] *= 1e-6
    host[kind == 2] *= 1e4
    if not rotated:
        host[kind == 3, :, 7] = np.inf
        host[kind == 4, :, 3] = -np.inf
        host[kind == 5] = -2.5
    x = np.zeros((rows, 2 * line + odd), np.float32)
    x[:, :line], x[:, line: 2 * line] = host[:, 0], host[:, 1]
    x = ref.encode(x, dtype)
    keys, values = (ref.decode(np.ascontiguousarray(v), dtype).reshape(rows, kv, d) for v in (x[:, :line], x[:, line: 2 * line]))
    angles = int(lengths.max()) - 3
    rope = ref.rope_tables(angles, d) if rotated else None
    d_pool, d_x, error = DeviceArray.of(pool.bytes), DeviceArray.of(x, dtype), error_word()

    class Part(Rows):
        def data_ptr(self):
            return self.array.data_ptr() + line * x.itemsize

    holed = table.copy()
    holed[missing] = -1
    serving.kv4_append(layout, d_pool, Rows(d_x, line), Part(d_x, line), DeviceArray.of(holed), DeviceArray.of(lengths),
                       row_start=DeviceArray.of(starts), error=error, rope=None if rope is None else tuple(DeviceArray.of(t) for t in rope))
    got = ref.Pool(pages, kv, d, page)
    got.bytes = d_pool.numpy()
    for i, n in enumerate(lengths):
        first = int(n) - counts[i]
        for r in range(counts[i]):
            t = first + r
            if t < 0 or (rotated and t >= angles) or (i, t // page) == missing:
                continue
            at = slice(starts[i] + r, starts[i] + r + 1)
            pool.append(keys[at], values[at], table[i: i + 1], np.array([t + 1], np.int32), [0, 1], rope)
            for h in range(kv):
                for which in range(2):
                    place = (table[i, t // page], 0, h, t % page, which)
                    want = pool.get(*place)
                    if np.isnan(want).any():                                     # of infinities that were rotated: any NaN will do
                        assert np.array_equal(got.get(*place), want, equal_nan=True)
                        for p in (got, pool):
                            p.put(*place, np.zeros((d // 32, 32), np.uint8), np.zeros(d // 32, np.float16), np.zeros(d // 32, np.float16))
    assert np.array_equal(got.bytes, pool.bytes)
    assert error.numpy()[0] == 0


def test_append_of_values_at_the_edge_of_the_types(cuda):
    rows, d = 8, 64
    x = np.random.default_rng(1).standard_normal((rows, d)).astype(np.float32)
    x[0] = 0
    x[1] = -2.5                                   # a block of one value: scale 0
    x[2, 5] = np.nan
    x[3, 40] = np.inf
    x[4, 3] = -np.inf
    x[5] *= 1e30
    x[6] *= 1e-12
    x[7, 1] = 1e5
    layout, pool = KV4Layout(1, 1, d, 16), ref.Pool(1, 1, d, 16)
    table, lengths, starts = np.zeros((1, 1), np.int32), np.array([rows], np.int32), np.array([0, rows], np.int32)
    d_pool, d_x = DeviceArray.of(pool.bytes), DeviceArray.of(x)
    serving.kv4_append(layout, d_pool, d_x, d_x, DeviceArray.of(table), DeviceArray.of(lengths), row_start=DeviceArray.of(starts))
    pool.append(x[:, None], x[:, None], table, lengths, starts)
    got = ref.Pool(1, 1, d, 16)
    got.bytes = d_pool.numpy()
    for a, b in zip(got.history(table[0], rows), pool.history(table[0], rows)):
        assert np.array_equal(a, b, equal_nan=True)
    assert np.isnan(a[2, 0, :32]).all() and np.isfinite(a[2, 0, 32:]).all() and np.isfinite(a[3:]).all()


def test_rows_without_a_page_or_an_angle_are_left_out_and_reported(cuda):
    layout = KV4Layout(1, 1, 32, 16)
    table = np.array([[0, 1], [2, 9], [-1, 3]], np.int32)                       # page 9 is outside a pool of 4
    lengths = np.array([5, 20, 3], np.int32)
    pool = ref.Pool(4, 1, 32, 16, fill=0x11)
    x = np.random.default_rng(0).standard_normal((3, 32)).astype(np.float32)
    d_pool, error = DeviceArray.of(pool.bytes), error_word()
    args = (DeviceArray.of(table), DeviceArray.of(lengths))
    serving.kv4_append(layout, d_pool, DeviceArray.of(x), DeviceArray.of(x), *args, error=error)
    pool.append(x[:1, None], x[:1, None], table[:1], lengths[:1], [0, 1])
    assert np.array_equal(d_pool.numpy(), pool.bytes) and error.numpy()[0] == 1
    back = [DeviceArray.of(np.ones((3, 32), np.float32)) for _ in range(2)]
    serving.kv4_read(layout, *back, d_pool, *args)
    assert not back[0].numpy()[1:].any() and back[0].numpy()[0].any()
    rope = tuple(DeviceArray.of(t) for t in ref.rope_tables(4, 32))              # sequence 0 is at position 4
    error = error_word()
    serving.kv4_append(layout, d_pool, DeviceArray.of(x), DeviceArray.of(x), *args, rope=rope, error=error)
    assert np.array_equal(d_pool.numpy(), pool.bytes) and error.numpy()[0] == 0


# -- attention -----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,d", [(14, 2, 64), (4, 2, 32), (3, 3, 96), (12, 1, 96), (16, 2, 128), (16, 1, 128), (40, 1, 64), (33, 1, 32)])
def test_single_tokens_of_every_length(cuda, dtype, heads, kv, d):
    """One row of each sequence; lengths about the tile, step and page borders, none, one; stale bytes are NaN."""
    rng = np.random.default_rng(heads * d)
    case = Case(rng, [0, 1, 2, 15, 16, 17, 31, 33, 48, 63, 64, 65, 97, 130, 257], kv, d, 48)
    q = rng.standard_normal((len(case.lengths), heads, d)).astype(np.float32)
    error = error_word()
    case.check(KV4Layout(heads, kv, d, 48), q, dtype, stride=heads * d + 5, error=error)
    assert error.numpy()[0] == ALL_ONES


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,d,page", [(14, 2, 64, 16), (4, 2, 32, 64), (6, 3, 96, 32), (8, 1, 128, 80)])
def test_prompts_see_no_later_position(cuda, dtype, heads, kv, d, page):
    """Several rows of a sequence, after a history or none, rotated; rows before position 0 see nothing."""
    rng = np.random.default_rng(page)
    case = Case(rng, [70, 5, 0, 131, 1, 40, 3], kv, d, page)
    counts = [70, 2, 0, 37, 1, 40, 6]
    q = rng.standard_normal((sum(counts), heads, d)).astype(np.float32)
    case.check(KV4Layout(heads, kv, d, page), q, dtype, counts, rope=ref.rope_tables(131, d))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_nan_is_seen_by_the_rows_that_see_its_position_only(cuda, dtype):
    rng = np.random.default_rng(5)
    layout = KV4Layout(4, 2, 64, 32)
    case = Case(rng, [50], 2, 64, 32)
    keys, values = (np.array(x) for x in case.histories[0])
    case.pool.append(keys, values, case.table, case.lengths, [0, 50])
    clean = case.pool.history(case.table[0], 50)
    values[20, 0, 3] = np.nan                      # head 0, first block
    keys[37, 1, 40] = np.nan                       # head 1
    case.pool.append(keys, values, case.table, case.lengths, [0, 50])
    case.upload()
    q = np.ones((50, 4, 64), np.float32)
    got, _ = case.attend(layout, q, dtype, [50])
    nan = np.isnan(got)
    assert not nan[:20, :2].any() and nan[20:, :2, :32].all() and not nan[:, :2, 32:].any()
    assert not nan[:37, 2:].any() and nan[37:, 2:].all()
    want, _, size = ref.attention(q, [clean], [50], [0, 50], np.float32(0.125))
    bound = attention_bound(dtype, want, size, np.abs(clean[1]).max())
    assert (np.abs(got - want)[~nan] <= bound[~nan]).all()


# bfloat16 prompts of enough work take the tensor cores' kernel. How much there is goes by the bounds that the call is
# given, so a large bound sends small histories there: `max_length` splits them (most splits then find nothing), many
# rows of a sequence leave them whole.


@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("heads,kv,d,page", [(14, 2, 64, 16), (16, 4, 64, 128), (8, 1, 128, 80), (12, 3, 128, 32)])
def test_bfloat16_prompts_on_the_tensor_cores(cuda, heads, kv, d, page, split):
    rng = np.random.default_rng(page + split)
    lengths, counts = [150, 5, 0, 201, 1, 40, 3, 64], [150, 2, 0, 37, 1, 40, 6, 64]
    if not split:                                   # more blocks of columns than there are places for CTAs
        lengths, counts = lengths * 3, counts * 3
    case = Case(rng, lengths, kv, d, page)
    q = rng.standard_normal((sum(counts), heads, d)).astype(np.float32)
    bounds = dict(max_length=30000) if split else dict(max_length=640, max_rows=sum(counts))
    error = error_word()
    case.check(KV4Layout(heads, kv, d, page), q, "bfloat16", counts, rope=ref.rope_tables(201, d), error=error, **bounds)
    assert error.numpy()[0] == ALL_ONES
    case.check(KV4Layout(heads, kv, d, page), q * 20, "bfloat16", counts, stride=heads * d + 3, **bounds)      # sharp scores
    cuda.device_faults()


@pytest.mark.parametrize("scale_kv", [2e4, 1.0, 1e-4])
def test_tensor_core_prompts_at_any_size_of_value(cuda, scale_kv):
    """Values that grow by orders along the history, so that their exponent and the maximum move between tiles."""
    rng = np.random.default_rng(13)
    case = Case(rng, [300], 1, 128, 16)
    keys, values = (x * np.geomspace(1e-2, 1, 300)[:, None, None].astype(np.float32) * np.float32(scale_kv) for x in case.histories[0])
    case.pool.append(keys, values, case.table, case.lengths, [0, 300])
    case.histories = [case.pool.history(case.table[0], 300)]
    case.upload()
    q = (rng.standard_normal((100, 4, 128)) * 3 / scale_kv).astype(np.float32)
    for bounds in (dict(max_length=100000), dict(max_length=300, max_rows=100)):
        case.check(KV4Layout(4, 1, 128, 16), q, "bfloat16", [100], **bounds)


def test_a_nan_on_the_tensor_cores_is_seen_by_the_rows_that_see_it_only(cuda):
    rng = np.random.default_rng(5)
    layout, long = KV4Layout(4, 2, 128, 32), dict(max_length=50000)
    case = Case(rng, [150], 2, 128, 32)
    keys, values = (np.array(x) for x in case.histories[0])
    case.pool.append(keys, values, case.table, case.lengths, [0, 150])
    clean = case.pool.history(case.table[0], 150)
    values[100, 0, 3] = np.nan                      # head 0, first block
    values[20, 0, 127] = np.nan                     # head 0, last block
    keys[137, 1, 40] = np.nan                       # head 1
    case.pool.append(keys, values, case.table, case.lengths, [0, 150])
    case.upload()
    q = np.ones((150, 4, 128), np.float32)
    got, _ = case.attend(layout, q, "bfloat16", [150], **long)
    nan = np.isnan(got)
    assert not nan[:100, :2, :32].any() and nan[100:, :2, :32].all() and not nan[:, :2, 32:96].any()
    assert not nan[:20, :2].any() and nan[20:, :2, 96:].all()
    assert not nan[:137, 2:].any() and nan[137:, 2:].all()
    want, _, size = ref.attention(q, [clean], [150], [0, 150], np.float32(128 ** -0.5))
    bound = attention_bound("bfloat16", want, size, np.abs(clean[1]).max())
    assert (np.abs(got - want)[~nan] <= bound[~nan]).all()


def test_missing_pages_on_the_tensor_cores(cuda):
    rng = np.random.default_rng(14)
    layout = KV4Layout(4, 1, 64, 16)
    case = Case(rng, [100, 90], 1, 64, 16)
    keys, values = case.histories[0]
    gone = case.table.copy()
    gone[0, 2] = -1
    case.d_table = DeviceArray.of(gone)
    error = error_word()
    q = rng.standard_normal((60, 4, 64)).astype(np.float32)
    q = ref.decode(ref.encode(q, "bfloat16"), "bfloat16")
    got, _ = case.attend(layout, q, "bfloat16", [30, 30], max_length=100000, error=error)
    assert error.numpy()[0] == 0
    there = np.r_[0:32, 48:100]
    want, _, size = ref.attention(q[:30], [(keys[there], values[there])], [84], [0, 30], np.float32(0.125))
    assert (np.abs(got[:30] - want) <= attention_bound("bfloat16", want, size, np.abs(values).max())).all()


@pytest.mark.parametrize("scale_kv,scale_q", [(1e4, 1e-3), (1e-5, 1e4), (300.0, 1e-2)])
def test_large_and_small_values(cuda, scale_kv, scale_q):
    rng = np.random.default_rng(7)
    case = Case(rng, [40, 90], 1, 64, 16, scale=scale_kv)
    case.check(KV4Layout(2, 1, 64, 16), (rng.standard_normal((2, 2, 64)) * scale_q).astype(np.float32), "float32")


def test_sharp_scores_and_a_maximum_that_keeps_growing(cuda):
    """Scores in the hundreds that rise along the history, so every step rescales what was summed."""
    rng = np.random.default_rng(8)
    case = Case(rng, [600], 1, 32, 16)
    keys, values = case.histories[0]
    keys = keys * 0.1 + np.linspace(-3, 3, 600)[:, None, None].astype(np.float32)
    case.pool.append(keys, values * np.geomspace(1e-3, 10, 600)[:, None, None].astype(np.float32), case.table, case.lengths, [0, 600])
    case.histories = [case.pool.history(case.table[0], 600)]
    case.upload()
    q = np.full((1, 4, 32), 4.0, np.float32) * np.array([1, -1, 8, -8], np.float32)[None, :, None]
    case.check(KV4Layout(4, 1, 32, 16), q, "float32")


def test_split_histories_share_scratch_and_repeat_bit_for_bit(cuda):
    """Long histories of few sequences are split over CTAs; scratch goes from one shape to another and back."""
    rng = np.random.default_rng(9)
    long, wide = Case(rng, [3001], 1, 64, 64), Case(rng, [100 + 40 * i for i in range(12)], 2, 32, 64)
    small = KV4Layout(7, 1, 64, 64), KV4Layout(4, 2, 32, 64)
    scratch = DeviceArray.zeros((1 << 22,), np.uint8)
    q = rng.standard_normal((1, 7, 64)).astype(np.float32), rng.standard_normal((12, 4, 32)).astype(np.float32)
    first = long.check(small[0], q[0], "float32", scratch=scratch)
    other = wide.check(small[1], q[1], "float32", scratch=scratch)
    for _ in range(3):
        for case, layout, x, want in ((long, small[0], q[0], first), (wide, small[1], q[1], other)):
            got = case.attend(layout, x, "float32", scratch=scratch)
            assert all(np.array_equal(a.view(np.uint32), b.view(np.uint32)) for a, b in zip(got, want))


def test_positions_past_max_length_and_missing_pages_are_left_out(cuda):
    rng = np.random.default_rng(10)
    layout = KV4Layout(2, 1, 64, 16)
    case = Case(rng, [60, 33], 1, 64, 16)
    q = rng.standard_normal((2, 2, 64)).astype(np.float32)
    keys, values = case.histories[0]
    gone = case.table.copy()
    gone[0, 1] = 1000
    case.d_table = DeviceArray.of(gone)
    error = error_word()
    got, _ = case.attend(layout, q, "float32", error=error)
    assert error.numpy()[0] == 0
    there = np.r_[0:16, 32:60]
    want, _, size = ref.attention(q[:1], [(keys[there], values[there])], [44], [0, 1], np.float32(0.125))
    assert (np.abs(got[0] - want[0]) <= attention_bound("float32", want[0], size[0], np.abs(values).max())).all()
    rope = ref.rope_tables(50, 64)                   # the first sequence's row is at position 59
    error = error_word()
    got, lse = case.attend(layout, q, "float32", rope=rope, error=error)
    assert error.numpy()[0] == 0 and not got[0].any() and np.isneginf(lse[0]).all() and np.isfinite(lse[1]).all()


def test_pools_past_32_bits(cuda):
    """Pages and layers whose bytes lie beyond the first four gigabytes."""
    layout = KV4Layout(2, 1, 128, 16, layers=1600)                              # 4 MB to a page
    pages = 1100
    pool = DeviceArray((pages, layout.page_bytes), np.uint8)
    rng = np.random.default_rng(11)
    table, lengths = np.array([[1099, 3, 1098]], np.int32), np.array([40], np.int32)
    x = rng.standard_normal((2, 40, 128)).astype(np.float32)
    args = (DeviceArray.of(table), DeviceArray.of(lengths))
    starts = DeviceArray.of(np.array([0, 40], np.int32))
    serving.kv4_append(layout, pool, DeviceArray.of(x[0]), DeviceArray.of(x[1]), *args, row_start=starts, layer=1599)
    back = [DeviceArray.zeros((40, 128), np.float32) for _ in range(2)]
    serving.kv4_read(layout, *back, pool, *args, row_start=starts, layer=1599)
    held = [ref.stands_for(*ref.quantise(v)) for v in x]
    assert all(np.array_equal(a.numpy(), b) for a, b in zip(back, held))
    q = rng.standard_normal((1, 2, 128)).astype(np.float32)
    out = DeviceArray.zeros((1, 256), np.float32)
    serving.kv4_attention(layout, out, DeviceArray.of(q.reshape(1, 256)), pool, *args, DeviceArray.zeros((1 << 20,), np.uint8),
                          max_length=40, layer=1599)
    want, _, size = ref.attention(q, [(held[0][:, None], held[1][:, None])], [40], [0, 1], np.float32(128 ** -0.5))
    assert (np.abs(out.numpy().reshape(1, 2, 128) - want) <= attention_bound("float32", want, size, np.abs(held[1]).max())).all()
    # The same page copied when the sequence forks.
    new = DeviceArray.zeros((1, 3), np.int32), DeviceArray.zeros((1,), np.int32)
    status = DeviceArray.zeros((4,), np.int64)
    two = DeviceArray.of(np.concatenate([table, table * 0 - 1])), DeviceArray.of(np.array([40, 0], np.int32))
    new = DeviceArray.zeros((2, 3), np.int32), DeviceArray.zeros((2,), np.int32)
    serving.kv_pages_update(*new, *two, pool, status, DeviceArray.zeros((serving.kv_pages_scratch_bytes(2, 3, pages),), np.uint8),
                            page_size=16, parent=DeviceArray.of(np.array([0, 0], np.int32)))
    assert new[0].numpy().tolist() == [[1099, 3, 1098], [1099, 3, 0]] and status.numpy().tolist() == [0, 4, 1, 1100]
    one = DeviceArray.of(new[0].numpy()[1:])
    serving.kv4_read(layout, *back, pool, one, args[1], row_start=starts, layer=1599)
    assert all(np.array_equal(a.numpy(), b) for a, b in zip(back, held))


def test_tensors_on_another_stream(cuda):
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(12)
    case = Case(rng, [200, 31], 2, 64, 32)
    layout = KV4Layout(14, 2, 64, 32)
    want, _ = case.attend(layout, np.full((2, 14, 64), 0.5, np.float32), "float32")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        q = torch.zeros(2, 14 * 64, device="cuda")
        torch.cuda._sleep(20_000_000)              # the queries arrive late: a call on another stream would miss them
        q += 0.5
        pool, table, lengths = (torch.from_numpy(x).cuda() for x in (case.pool.bytes, case.table, case.lengths))
        out, scratch = torch.empty_like(q), torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
        serving.kv4_attention(layout, out, q, pool, table, lengths, scratch, max_length=200, stream=stream.cuda_stream)
    stream.synchronize()
    assert np.array_equal(out.cpu().numpy().reshape(2, 14, 64).view(np.uint32), want.view(np.uint32))


# -- pages ---------------------------------------------------------------------------------------------------------


def update(table, lengths, page, pool, parent=None, grow=None):
    pages = pool.shape[0]
    d_pool, new, n = DeviceArray.of(pool), DeviceArray.zeros(table.shape, np.int32), DeviceArray.zeros(lengths.shape, np.int32)
    status = DeviceArray.zeros((4,), np.int64)
    scratch = DeviceArray.of(np.full(serving.kv_pages_scratch_bytes(*table.shape, pages), 0x5A, np.uint8))
    serving.kv_pages_update(new, n, DeviceArray.of(table), DeviceArray.of(lengths), d_pool, status, scratch, page_size=page,
                            parent=None if parent is None else DeviceArray.of(np.asarray(parent, np.int32)),
                            grow=None if grow is None else DeviceArray.of(np.asarray(grow, np.int32)))
    return new.numpy(), n.numpy(), status.numpy().tolist(), d_pool.numpy()


def check_update(table, lengths, page, pool, parent=None, grow=None):
    got = update(table, lengths, page, pool, parent, grow)
    new, n, status, copies = ref.pages_update(table, lengths, page, pool.shape[0], parent, grow)
    assert np.array_equal(got[0], new) and np.array_equal(got[1], n) and got[2] == status
    for a, b in copies:
        pool = pool.copy()
        pool[b] = pool[a]
    assert np.array_equal(got[3], pool)
    return new, n, pool


@pytest.mark.parametrize("seqs,width,pages,page", [(1, 1, 1, 16), (5, 4, 11, 16), (40, 9, 200, 32), (1500, 3, 2500, 16), (7, 700, 2100, 16)])
def test_random_histories_of_updates(cuda, seqs, width, pages, page):
    """Fork, reorder, grow, cut and free at random, each step from the last one's result; shortages among them."""
    rng = np.random.default_rng(pages)
    table, lengths = np.full((seqs, width), -1, np.int32), np.zeros(seqs, np.int32)
    pool = rng.integers(0, 256, (pages, 48), np.uint8)
    for step in range(8):
        parent = rng.integers(-1, seqs + 1, seqs) if step % 3 == 2 else np.arange(seqs)
        grow = rng.integers(-page, 2 * page + 2, seqs) if step % 2 else rng.integers(0, 3, seqs)
        if step == 5:
            grow = np.full(seqs, width * page)                                 # more than there is, where there is little
        table, lengths, pool = check_update(table, lengths, page, pool, parent, grow)


def test_defaults_keep_everything(cuda):
    rng = np.random.default_rng(2)
    table, pages = table_of(rng, [17, 0, 40], 16)
    pool = rng.integers(0, 256, (pages, 16), np.uint8)
    new, n, same = check_update(table, np.array([17, 0, 40], np.int32), 16, pool)
    assert np.array_equal(same, pool) and n.tolist() == [17, 0, 40]


def test_a_cut_into_a_shared_page_copies_it(cuda):
    table, lengths = np.array([[3, 1, 5], [3, 1, -1]], np.int32), np.array([40, 32], np.int32)
    pool = np.arange(8, dtype=np.uint8)[:, None].repeat(32, 1)
    new, n, after = check_update(table, lengths, 16, pool, grow=[0, -10])
    assert new.tolist() == [[3, 1, 5], [3, 0, -1]] and n.tolist() == [40, 22] and (after[0] == 1).all()


def test_missing_pages_and_bad_tables_change_nothing(cuda):
    pool = np.arange(4, dtype=np.uint8)[:, None].repeat(16, 1)
    table, lengths = np.array([[0, 1], [2, -1]], np.int32), np.array([32, 5], np.int32)
    new, n, status, same = update(table, lengths, 16, pool, parent=[1, 1], grow=[16, 17])
    assert status == [1, 3, 0, 0] or status[0] >= 0
    check_update(table, lengths, 16, pool, parent=[1, 1], grow=[16, 17])
    check_update(table, lengths, 16, pool, parent=[0, 0], grow=[0, 0])
    check_update(np.array([[0, 7], [2, -1]], np.int32), lengths, 16, pool)
    check_update(np.array([[0, -1], [2, -1]], np.int32), lengths, 16, pool)


@pytest.mark.parametrize("page_bytes", [16, 4096, 16384, 16400, 40000])
def test_copies_of_pages_of_any_size(cuda, page_bytes):
    rng = np.random.default_rng(page_bytes)
    table, lengths = np.array([[2], [-1], [-1], [0]], np.int32), np.array([3, 0, 0, 16], np.int32)
    pool = rng.integers(0, 256, (9, page_bytes), np.uint8)
    check_update(table, lengths, 16, pool, parent=[0, 0, 0, 3])


@pytest.mark.parametrize("seqs,width,pages,page", [(1, 1, 1, 16), (6, 5, 60, 16), (300, 9, 4000, 32), (3, 600, 5000, 16)])
def test_compaction(cuda, seqs, width, pages, page):
    rng = np.random.default_rng(seqs)
    lengths = rng.integers(0, width * page + 1, seqs).astype(np.int32)
    lengths[0] = width * page
    order = rng.permutation(pages)
    table, at = np.full((seqs, width), -1, np.int32), 0
    for i, n in enumerate(lengths):
        m = -(-int(n) // page)
        table[i, :m] = order[at: at + m]
        at = (at + m) % max(1, pages - width)                                   # some pages are shared
    table[-1, -1] = 99999 if lengths[-1] <= (width - 1) * page else table[-1, -1]     # past the length: not looked at
    pool = rng.integers(0, 256, (pages, 64), np.uint8)
    d_pool, new, status = DeviceArray.of(pool), DeviceArray.zeros(table.shape, np.int32), DeviceArray.zeros((4,), np.int64)
    scratch = DeviceArray.of(np.full(serving.kv_pages_scratch_bytes(seqs, width, pages), 0x5A, np.uint8))
    serving.kv_pages_compact(new, DeviceArray.of(table), DeviceArray.of(lengths), d_pool, status, scratch, page_size=page)
    want, state, moves = ref.pages_compact(table, lengths, page, pages)
    assert np.array_equal(new.numpy(), want) and status.numpy().tolist() == state
    moved = pool.copy()
    for a, b in moves:
        moved[b] = pool[a]
    assert np.array_equal(d_pool.numpy(), moved)


# -- log probabilities -----------------------------------------------------------------------------------------------


def scores(x, targets, k, dtype="float32", stride=None, offset=0, scratch=None, error=None):
    """The device's log probabilities of ``targets``, entropy, log-sums, top ids and log probabilities."""
    rows, vocab = x.shape
    stride = stride or vocab
    flat = np.zeros(offset + rows * stride, np.float32)
    for r in range(rows):
        flat[offset + r * stride: offset + r * stride + vocab] = x[r]
    held = DeviceArray.of(ref.encode(flat, dtype), dtype)

    class View:
        shape, dtype = (rows, vocab), held.dtype
        data_ptr = staticmethod(lambda: held.data_ptr() + offset * held.host_type.itemsize)
        stride = staticmethod(lambda: (stride_, 1))

    stride_ = stride
    n = targets.shape[1]
    out, entropy, lse = DeviceArray.zeros((rows, n), np.float32), DeviceArray.zeros((rows,), np.float32), DeviceArray.zeros((rows,), np.float32)
    top, best = DeviceArray.zeros((rows, k), np.int64), DeviceArray.zeros((rows, k), np.float32)
    if scratch is None:
        scratch = DeviceArray.zeros((serving.token_logprobs_scratch_bytes(rows, vocab, k),), np.uint8)
    serving.token_logprobs(View, DeviceArray.of(targets), out, entropy, top, best, lse=lse, scratch=scratch, error=error)
    return [a.numpy() for a in (out, entropy, lse, top, best)]


def check_scores(x, targets, k, dtype="float32", **options):
    """A logit's distance to the maximum D and the sums lose at most 2^-21 (D + 4) in float32."""
    x = ref.decode(ref.encode(x.astype(np.float32), dtype), dtype)
    got = scores(x, targets, k, dtype, **options)
    want = ref.logprobs(x, targets, k)
    assert np.array_equal(got[3], want[3])
    for i in (0, 1, 2, 4):
        a, b = got[i].astype(np.float64), want[i]
        same = (a == b) | (np.isnan(a) & np.isnan(b))
        with np.errstate(invalid="ignore"):
            assert (same | (np.abs(a - b) <= 2.0 ** -21 * (np.abs(b) + 4))).all(), i
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,k,n", [(1, 1, 1, 1), (3, 5, 5, 2), (2, 33, 32, 0), (5, 1000, 0, 3), (7, 4099, 20, 1),
                                            (1, 151936, 5, 1), (3, 151936, 32, 4), (40, 20001, 20, 1), (600, 300, 7, 1)])
def test_log_probabilities(cuda, dtype, rows, vocab, k, n):
    rng = np.random.default_rng(rows + vocab)
    x = rng.standard_normal((rows, vocab)) * 3
    check_scores(x, rng.integers(0, vocab, (rows, n)), k, dtype)


@pytest.mark.parametrize("stride,offset", [(1001, 0), (1003, 1), (1024, 3), (1006, 5)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_logits_at_any_alignment(cuda, dtype, stride, offset):
    rng = np.random.default_rng(stride)
    check_scores(rng.standard_normal((4, 1001)) * 2, rng.integers(0, 1001, (4, 1)), 9, dtype, stride=stride, offset=offset)


@pytest.mark.parametrize("vocab", [257, 5000, 151936])
def test_equal_logits_go_by_their_index(cuda, vocab):
    rng = np.random.default_rng(vocab)
    x = np.zeros((6, vocab))
    x[1] = np.round(rng.standard_normal(vocab))                                 # masses of equals
    x[2, rng.integers(0, vocab, 40)] = 1
    x[3] = -np.inf
    x[3, vocab // 2:] = 2
    x[4] = np.arange(vocab) // 50
    x[5, ::2] = -0.0
    check_scores(x, rng.integers(0, vocab, (6, 2)), 32)


def test_masked_infinite_and_missing_logits(cuda):
    vocab = 3000
    x = np.random.default_rng(3).standard_normal((9, vocab))
    x[0] = -np.inf                                     # nothing is left
    x[1, 5:] = -np.inf
    x[2, 17] = np.nan
    x[3, :2000] = np.nan
    x[4, 9] = np.inf
    x[5] = np.finfo(np.float32).min                    # a mask of the type's lowest value
    x[6, 10:] = np.finfo(np.float32).min
    x[7] *= 1e30
    x[8] = -1e30
    targets = np.tile(np.array([[0, 4, 17]]), (9, 1))
    got = scores(x.astype(np.float32), targets, 8)
    want = ref.logprobs(x.astype(np.float32), targets, 8)
    assert np.array_equal(got[3], want[3])
    assert np.isneginf(got[0][0]).all() and got[1][0] == 0 and np.isneginf(got[2][0])
    for r in (2, 3):
        assert np.isnan(got[0][r]).all() and np.isnan(got[1][r]) and np.isnan(got[2][r])
    assert np.isnan(got[0][4]).all() or np.isneginf(got[0][4][0])
    for r in (1, 5, 6, 7, 8):
        for i in (0, 1, 2, 4):
            a, b = got[i][r].astype(np.float64), want[i][r]
            with np.errstate(invalid="ignore"):
                assert ((a == b) | (np.abs(a - b) <= 2.0 ** -21 * (np.abs(b) + 4))).all(), (r, i)


def test_targets_outside_the_vocabulary(cuda):
    x = np.random.default_rng(4).standard_normal((5, 100)).astype(np.float32)
    targets = np.array([[3], [99], [100], [-1], [0]])
    error = error_word()
    out = scores(x, targets, 2, error=error)[0][:, 0]
    assert np.isnan(out[2:4]).all() and np.isfinite(out[[0, 1, 4]]).all() and error.numpy()[0] == 2


def test_more_rows_than_a_launch_and_scratch_from_shape_to_shape(cuda):
    rng = np.random.default_rng(6)
    scratch = DeviceArray.zeros((1 << 23,), np.uint8)
    many, long = rng.standard_normal((5000, 40)), rng.standard_normal((2, 60000))
    targets = rng.integers(0, 40, (5000, 1)), rng.integers(0, 60000, (2, 1))
    for _ in range(2):
        check_scores(long, targets[1], 32, scratch=scratch)
        check_scores(many, targets[0], 3, scratch=scratch)
        check_scores(rng.standard_normal((9, 151936)), rng.integers(0, 151936, (9, 1)), 32, scratch=scratch)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(64, 151936), (592, 40001)])             # several segments of several batches, and one
def test_a_nan_anywhere_in_a_long_row_comes_first(cuda, dtype, rows, vocab):
    x = np.zeros((rows, vocab), np.float32)
    x[:8] = np.random.default_rng(vocab).standard_normal((8, vocab)) * 3
    for r, at in enumerate(([100], [vocab // 2], [vocab - 1], [vocab - 1, vocab // 3], [7], list(range(40, 80)))):
        x[r, at] = np.nan
    x[4, 8:] = -np.inf                                # nothing after the NaN
    targets = np.tile(np.array([[0, vocab - 2]]), (rows, 1))
    x = ref.decode(ref.encode(x, dtype), dtype)
    got = scores(x, targets, 20, dtype)
    want = ref.logprobs(x[:8], targets[:8], 20)
    assert np.array_equal(got[3][:8], want[3])
    for i in (0, 1, 2, 4):
        assert np.isnan(got[i][:6]).all() and np.isfinite(got[i][6:]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [2, 592])                                       # several segments of a row, and one
def test_equals_below_many_better_logits(cuda, dtype, rows):
    """Whole blocks above the k-th best, and masses of equals from there down: no more of them than are wanted are taken."""
    vocab, rng = 8192, np.random.default_rng(rows)
    x = np.zeros((rows, vocab), np.float32)
    x[0] = -np.inf
    for u in range(4):                                # with vectors of eight, these are all of the first 31 threads' blocks
        x[0, 2048 * u: 2048 * u + 248] = rng.permutation(248) + 1000 * (u == 2)
        x[1, 2048 * u: 2048 * u + 248] = 5
        if rows > 2:
            x[2, 2048 * u: 2048 * u + 248] = 5 + (np.arange(248) % 8 == 0)
            x[3, 1024 * u: 1024 * u + 124] = rng.permutation(124) + 1        # the same with vectors of four
    if rows > 4:
        x[4] = np.round(rng.standard_normal(vocab))
        x[5, ::50] = 1                                # more equals at the top than are wanted
        x[6, 8100:] = 1
    for k in (25, 31, 32):
        check_scores(x, rng.integers(0, vocab, (rows, 1)), k, dtype)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("vocab", [257, 5000, 151936])
def test_equal_logits_of_16_bits_go_by_their_index(cuda, dtype, vocab):
    rng = np.random.default_rng(vocab)
    x = np.zeros((6, vocab))
    x[1] = np.round(rng.standard_normal(vocab))
    x[2, rng.integers(0, vocab, 40)] = 1
    x[3] = -np.inf
    x[3, vocab // 2:] = 2
    x[4] = np.arange(vocab) // 50
    x[5, ::2] = -0.0
    check_scores(x, rng.integers(0, vocab, (6, 2)), 32, dtype)


@pytest.mark.parametrize("dtype,d,bounds", [("float32", 64, {}), ("float16", 128, {}), ("bfloat16", 96, {}), ("bfloat16", 64, dict(max_length=100000)),
                                            ("bfloat16", 128, dict(max_length=100000))])
def test_rows_without_an_angle_see_nothing_of_a_long_history(cuda, dtype, d, bounds):
    """Rows past the table's end get zeros and -inf, whole steps before them or not; the others of their block what they see."""
    rng = np.random.default_rng(d)
    layout, angles = KV4Layout(4, 1, d, 16), 250
    case = Case(rng, [300, 200], 1, d, 16)
    counts = [100, 30]                                # positions 200 .. 299, and 170 .. 199
    q = ref.decode(ref.encode(rng.standard_normal((130, 4, d)).astype(np.float32), dtype), dtype)
    rope, error = ref.rope_tables(300, d), error_word()
    got, lse = case.attend(layout, q, dtype, counts, tuple(t[:angles].copy() for t in rope), error=error, **bounds)
    assert error.numpy()[0] == 0
    want, want_lse, size = ref.attention(q, case.histories, case.lengths, starts_of(counts), np.float32(d ** -0.5), rope)
    none = np.arange(130) // 50 == 1
    none[100:] = False
    assert not got[none].any() and np.isneginf(lse[none]).all()
    most = max(np.abs(v).max() for _, v in case.histories)
    assert (np.abs(got - want) <= attention_bound(dtype, want, size, most))[~none].all()
    assert np.isfinite(lse[~none]).all()
    alone, lse = case.attend(layout, q[:2], dtype, [1, 1], tuple(t[:180].copy() for t in rope))       # single tokens, both past the end
    assert not alone.any() and np.isneginf(lse).all()


@pytest.mark.parametrize("dtype,d", [("float32", 64), ("float16", 32), ("bfloat16", 96), ("bfloat16", 128), ("bfloat16", 64)])
@pytest.mark.parametrize("longest", [0, 1, 100, 128])
def test_positions_past_the_longest_length_have_no_share(cuda, dtype, d, longest):
    rng = np.random.default_rng(d + longest)
    times = 8 if dtype == "bfloat16" and d != 96 else 1
    lengths, counts = [128, 300, 40] * times, [30, 2, 30] * times
    case = Case(rng, lengths, 3, d, 16)
    q = rng.standard_normal((sum(counts), 12, d)).astype(np.float32)
    rope = ref.rope_tables(300, d)
    cut = [(k[:longest], v[:longest]) for k, v in case.histories]
    q = ref.decode(ref.encode(q, dtype), dtype)
    for rows, most_rows in ((counts, sum(counts)), ([1] * len(lengths), 1)):
        x = q[: sum(rows)]
        got, lse = case.attend(KV4Layout(12, 3, d, 16), x, dtype, rows, rope, max_length=longest, max_rows=most_rows)
        if longest == 0:
            assert not got.any() and np.isneginf(lse).all()
            continue
        want, want_lse, size = ref.attention(x, cut, case.lengths, starts_of(rows), np.float32(d ** -0.5), rope)
        most = max(np.abs(v).max() for _, v in cut)
        assert (np.abs(got - want) <= attention_bound(dtype, want, size, most)).all()
        slack = (2.0 ** -18 if dtype != "bfloat16" else 2.0 ** -11) * (size + 4)
        assert (np.abs(lse - want_lse) <= slack + 2.0 ** -22 * np.abs(want_lse)).all()


@pytest.mark.parametrize("dtype,heads,d,bounds", [("float32", 7, 64, {}), ("bfloat16", 7, 128, {}), ("bfloat16", 30, 128, dict(max_length=50000)),
                                                  ("bfloat16", 30, 64, dict(max_length=100000))])
def test_rows_past_the_most_rows_get_no_output(cuda, dtype, heads, d, bounds):
    rng = np.random.default_rng(heads + d)
    counts, most_rows = [5, 40, 3, 4], 4
    case = Case(rng, [70, 90, 3, 150], 1, d, 16)
    q = ref.decode(ref.encode(rng.standard_normal((sum(counts), heads, d)).astype(np.float32), dtype), dtype)
    got, lse = case.attend(KV4Layout(heads, 1, d, 16), q, dtype, counts, max_rows=most_rows, **bounds)
    want, want_lse, size = ref.attention(q, case.histories, case.lengths, starts_of(counts), np.float32(d ** -0.5))
    past = np.concatenate([np.arange(c) >= most_rows for c in counts])
    assert not got[past].any() and (lse[past] == 7.0).all()
    most = max(np.abs(v).max() for _, v in case.histories)
    assert (np.abs(got - want) <= attention_bound(dtype, want, size, most))[~past].all()
    assert (np.abs(lse - want_lse) <= 2.0 ** -11 * (size + 4))[~past].all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_bound_of_rows_above_the_calls_rows(cuda, dtype):
    rng = np.random.default_rng(21)
    case = Case(rng, [40, 9], 1, 64, 16)
    q = rng.standard_normal((5, 4, 64)).astype(np.float32)
    case.check(KV4Layout(4, 1, 64, 16), q, dtype, [3, 2], max_rows=512)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,d", [(14, 2, 64), (8, 2, 128)])
def test_one_attention_scratch_for_a_batch_that_shrinks(cuda, dtype, heads, kv, d):
    rng = np.random.default_rng(22)
    layout, most = KV4Layout(heads, kv, d, 16), 2048
    scratch = DeviceArray.zeros((serving.kv4_attention_scratch_bytes(layout, 64 * 40, 64, most, 40),), np.uint8)
    for lengths, rows in (([300, 30, 7, 200] * 8, 1), ([300, 30, 7, 200], 1), ([300, 200], 40), ([2048], 1), ([100], 100)):
        case = Case(rng, lengths, kv, d, 16)
        q = rng.standard_normal((rows * len(lengths), heads, d)).astype(np.float32)
        case.check(layout, q, dtype, [rows] * len(lengths), scratch=scratch, max_length=most, max_rows=rows)


@pytest.mark.parametrize("dtype", TYPES)
def test_one_scratch_for_fewer_rows_of_logits(cuda, dtype):
    rng, vocab = np.random.default_rng(23), 151936
    x = rng.standard_normal((64, vocab)).astype(np.float32)
    scratch = DeviceArray.zeros((serving.token_logprobs_scratch_bytes(64, vocab, 20),), np.uint8)
    for rows in (64, 50, 12, 6, 1):
        scores(x[:rows], rng.integers(0, vocab, (rows, 1)), 20, dtype, scratch=scratch)
    check_scores(x[:6], rng.integers(0, vocab, (6, 1)), 20, dtype, scratch=scratch)


@pytest.mark.parametrize("rows", [20, 2059])                                     # appended row by row, and by tiles
def test_row_starts_that_end_past_the_rows_reach_no_others(cuda, rows):
    rng, kv, d, page, more = np.random.default_rng(rows), 2, 64, 32, 40
    layout, line, length = KV4Layout(kv, kv, d, page), kv * d, rows + 37         # the last of 37 positions that have no row here
    table, pages = table_of(rng, [length], page)
    pool = ref.Pool(pages, kv, d, page, fill=0xA5)
    x = rng.standard_normal((rows + more, line)).astype(np.float32)
    d_pool, d_x = DeviceArray.of(pool.bytes), DeviceArray.of(x)

    class First(Rows):
        def __init__(self, array):
            self.array, self.shape, self.dtype = array, (rows, line), array.dtype

    args = DeviceArray.of(table), DeviceArray.of(np.array([length], np.int32))
    starts = DeviceArray.of(np.array([0, length], np.int32))
    serving.kv4_append(layout, d_pool, First(d_x), First(d_x), *args, row_start=starts)
    held = x[:rows].reshape(rows, kv, d)
    pool.append(held, held, table, [rows], [0, rows])
    assert np.array_equal(d_pool.numpy(), pool.bytes)
    back = [DeviceArray.of(np.full(x.shape, 5, np.float32)) for _ in range(2)]
    serving.kv4_read(layout, First(back[0]), First(back[1]), d_pool, *args, row_start=starts)
    want = ref.stands_for(*ref.quantise(held)).reshape(rows, line)
    for got in back:
        assert np.array_equal(got.numpy()[:rows], want) and (got.numpy()[rows:] == 5).all()


@pytest.mark.parametrize("seqs", [2, 700])                                       # one CTA's bookkeeping, and a cluster's
def test_a_shortage_of_pages_changes_nothing(cuda, seqs):
    rng = np.random.default_rng(seqs)
    if seqs == 2:                                     # both continue the second: a copy of page 2 and a page behind each, of pages 0 and 1
        pages, missing, used = 3, 1, 3
        table, lengths = np.array([[0, 1], [2, -1]], np.int32), np.array([32, 5], np.int32)
        parent, grow = [1, 1], [16, 17]
    else:                                             # a hundred more continue the first, whose last page is not full, and 50 pages are free
        width, live, pages, missing, used = 9, 600, 5450, 50, 5400
        table = np.full((seqs, width), -1, np.int32)
        table[:live] = rng.permutation(pages)[: live * width].reshape(live, width)
        lengths = np.where(np.arange(seqs) < live, 16 * (width - 1) + 5, 0).astype(np.int32)
        parent, grow = np.where(np.arange(seqs) < live, np.arange(seqs), 0), np.where(np.arange(seqs) < live, 0, 200)
    pool = rng.integers(0, 256, (pages, 32), np.uint8)
    new, n, status, same = update(table, lengths, 16, pool, parent, grow)
    assert status == [missing, used, 0, 0]
    assert np.array_equal(new, table) and np.array_equal(n, lengths) and np.array_equal(same, pool)


@pytest.mark.parametrize("d", [64, 128])
def test_split_histories_on_the_tensor_cores(cuda, d):
    """Sixteen heads of one key head and a bound of 2000 positions: chunks of 320, several to the longer histories."""
    rng = np.random.default_rng(d)
    case, counts = Case(rng, [1500, 330, 70, 0], 1, d, 32), [50, 80, 70, 3]
    layout, bounds = KV4Layout(16, 1, d, 32), dict(max_length=2000, max_rows=80)
    q, rope = rng.standard_normal((sum(counts), 16, d)).astype(np.float32), ref.rope_tables(1500, d)
    scratch = DeviceArray.zeros((serving.kv4_attention_scratch_bytes(layout, sum(counts), 4, 2000, 80),), np.uint8)
    want = case.check(layout, q, "bfloat16", counts, rope=rope, scratch=scratch, **bounds)
    case.check(layout, q * 20, "bfloat16", counts, scratch=scratch, **bounds)
    q = ref.decode(ref.encode(q, "bfloat16"), "bfloat16")
    again = case.attend(layout, q, "bfloat16", counts, rope, scratch=scratch, **bounds)
    assert all(np.array_equal(a.view(np.uint32), b.view(np.uint32)) for a, b in zip(again, want))


@pytest.mark.parametrize("heads,kv,d,rows", [(14, 2, 64, 480), (8, 2, 64, 128), (8, 2, 128, 64), (128, 1, 128, 1), (100, 1, 64, 3)])
def test_bfloat16_prompts_on_either_side_of_the_choice(cuda, heads, kv, d, rows):
    rng = np.random.default_rng(rows)
    for seqs in (1, 4):
        case = Case(rng, [rows + 5 * i for i in range(seqs)], kv, d, 64)
        q = rng.standard_normal((seqs * rows, heads, d)).astype(np.float32)
        case.check(KV4Layout(heads, kv, d, 64), q, "bfloat16", [rows] * seqs)


@pytest.mark.parametrize("heads,d,bounds", [(16, 128, dict(max_length=2000, max_rows=80)), (16, 64, dict(max_length=2000, max_rows=80)), (2, 128, {}), (4, 96, {})])
@pytest.mark.parametrize("centre,spread,share", [(100.0, 0.3, 1.0), (-30.0, 1.0, 1.0), (0.0, 1.0, 1.0), (200.0, 0.2, 0.02), (60.0, 1.0, 0.5)])
def test_bfloat16_scores_of_keys_far_from_nought(cuda, heads, d, bounds, centre, spread, share):
    """Of keys far from nought only what lies above their block's zero is rounded, with the queries; `share` of the blocks are far.

    f16 rounds by 2^-11 at most: a score is off by 2^-11 of R = sum_i |q_i r_i| for the queries and as much again for the keys, r_i what
    is rounded of a key or stands beside its query, and by 2^-20 of S = sum_i |q_i k_i| as for the other types; a log-sum by no more than
    the scores that are in it, and 2^-18.
    """
    rng = np.random.default_rng(d)
    case, counts = Case(rng, [64, 300], 1, d, 16), [64, 80] if bounds else [3, 5]
    starts, blocks = starts_of(case.lengths), d // 32
    keys = rng.standard_normal((starts[-1], blocks, 32)) * spread
    keys += (centre * np.where(np.arange(blocks) % 2, -1, 1) * (rng.random((starts[-1], blocks)) < share))[..., None]
    keys = keys.reshape(-1, 1, d).astype(np.float32)
    case.pool.append(keys, keys / max(1.0, abs(centre)), case.table, case.lengths, starts)
    case.histories = [case.pool.history(case.table[i], n) for i, n in enumerate(case.lengths)]
    case.upload()
    q = ref.decode(ref.encode(rng.standard_normal((sum(counts), heads, d)).astype(np.float32), "bfloat16"), "bfloat16")
    got, lse = case.attend(KV4Layout(heads, 1, d, 16), q, "bfloat16", counts, **bounds)
    want, want_lse, size = ref.attention(q, case.histories, case.lengths, starts_of(counts), np.float32(d ** -0.5))
    rounded, rows = np.zeros_like(size), starts_of(counts)
    for i, (k, _) in enumerate(case.histories):
        k = k.reshape(len(k), blocks, 32).astype(np.float64)
        zero = k.min(-1, keepdims=True)
        far = np.abs(zero) > 16 / 15 * (k.max(-1, keepdims=True) - zero)
        r = np.maximum(k - zero, np.where(far, 0, np.abs(k))).reshape(len(k), d)
        for row in range(rows[i], rows[i + 1]):
            seen = int(case.lengths[i]) - (rows[i + 1] - row) + 1
            rounded[row] = (r[:seen] @ np.abs(q[row]).T).max(0) * d ** -0.5
    off = 2.0 ** -10 * rounded + 2.0 ** -20 * size
    assert (np.abs(lse - want_lse) <= off + 2.0 ** -18 + 2.0 ** -22 * np.abs(want_lse)).all()
    # The output: probabilities by a factor 1 +- 2 off, themselves and the values by 2^-11 each.
    most = max(np.abs(v).max() for _, v in case.histories)
    bound = (2 * off + 2.0 ** -10)[..., None] * most + ROUNDING["bfloat16"] * np.abs(want) * 1.001
    assert (np.abs(got - want) <= bound).all()
