"""Adapters, beam selection and reordering of states on the GPU against their plain forms in 64 bits (``requests_ref``).

Adapters may differ by the float32 sums' bound, which the plain form gives, and by half a step of the output's type. Beams are
equal where the totals lie further apart than 4e-6 + 2^-22 of a total: a log-sum's float32 sums of a row that is cut into segments
lose less than 32 roundings of 2^-24 of the sum and 2^-21 for its exponentials. States are moved, hence equal.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from nanocompile_b200 import runtime, serving
from nanocompile_b200.serving import DeviceArray, LoraBatch, LoraLayout
from tests import requests_ref as ref
from tests.serving_ref import BF16, decode, encode

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", BF16]
ROUNDING = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, BF16: 2.0 ** -8}
ALL_ONES = np.uint64(0xFFFFFFFFFFFFFFFF)


class View:
    """A device array looked at with other sizes, strides or a later beginning (in elements)."""

    def __init__(self, array, shape, strides, skip=0):
        self.array, self.shape, self.strides, self.skip, self.dtype = array, tuple(shape), tuple(strides), skip, array.dtype

    def data_ptr(self):
        return self.array.data_ptr() + self.skip * self.array.host_type.itemsize

    def stride(self):
        return self.strides

    def is_contiguous(self):
        return False


def device(host, dtype):
    return DeviceArray.of(encode(host, dtype), dtype if dtype == BF16 else None)


def strided(host, dtype, stride, skip):
    """Rows of ``host`` at another stride, ``skip`` elements into their buffer; the view and the buffer."""
    rows, line = host.shape
    room = np.full(skip + max(rows, 1) * stride, 77, np.float32)
    for i in range(rows):
        room[skip + i * stride: skip + i * stride + line] = host[i]
    array = device(room, dtype)
    return View(array, (rows, line), (stride, 1), skip), array


def rounded(values, dtype):
    return decode(encode(np.asarray(values, np.float32), dtype), dtype)


def error_word():
    return DeviceArray.of(np.array([ALL_ONES]))


class Adapted:
    """A batch of sequences with adapters, on the host and the device."""

    def __init__(self, seed, dtype, wtype, inputs, widths, rank, slots, adapters, counts, ranks=None, scales=True, base=True, tail=0):
        rng = np.random.default_rng(seed)
        self.dtype, self.wtype, self.widths, self.rank = dtype, wtype, widths, rank
        self.adapters = np.asarray(adapters, np.int32)
        self.row_start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        rows = int(self.row_start[-1]) + tail
        self.x = rounded(rng.standard_normal((rows, inputs)), dtype)
        self.a = rounded(rng.standard_normal((slots, len(widths) * rank, inputs)) * inputs ** -0.5, wtype)
        self.b = rounded(rng.standard_normal((slots, sum(widths), rank)) * 0.2, wtype)
        self.base = rounded(rng.standard_normal((rows, sum(widths))), dtype) if base else None
        self.ranks = None if ranks is None else np.asarray(ranks, np.int32)
        self.scales = rng.uniform(0.5, 3, slots).astype(np.float32) if scales else None
        self.layout, self.batch = LoraLayout(inputs, widths, rank), LoraBatch(rows, len(counts), slots)

    def upload(self):
        opt = lambda v: None if v is None else DeviceArray.of(v)                                     # noqa: E731
        self.d_a, self.d_b = device(self.a, self.wtype), device(self.b, self.wtype)
        self.d_ranks, self.d_scales = opt(self.ranks), opt(self.scales)
        self.plan = DeviceArray((self.batch.plan_bytes,), np.uint8)
        self.d_adapters, self.d_start = DeviceArray.of(self.adapters), DeviceArray.of(self.row_start)

    def run(self, x=None, base=None, out=None, error=None, by_row=False, stream=0):
        self.upload()
        self.d_x = x or device(self.x, self.dtype)
        self.d_base = base if base is not None else None if self.base is None else device(self.base, self.dtype)
        self.d_out = out or device(np.full((self.batch.rows, sum(self.widths)), 55), self.dtype)
        serving.lora_plan(self.batch, self.plan, self.d_adapters, row_start=None if by_row else self.d_start, error=error, stream=stream)
        serving.lora_project(self.layout, self.batch, self.d_out, self.d_x, self.d_a, self.d_b, self.plan, base=self.d_base,
                             ranks=self.d_ranks, scales=self.d_scales, stream=stream)
        return self

    def check(self, got=None):
        got = decode(self.d_out.numpy(), self.dtype) if got is None else got
        n = int(self.row_start[-1])
        want, bound = ref.lora(self.x, self.a, self.b, self.widths, self.rank, self.adapters, self.row_start, self.base, self.ranks, self.scales)
        # The product with the scale and the sum with base round once more each in float32; the output's own type last.
        bound = bound + 2.0 ** -23 * np.abs(want) + ROUNDING[self.dtype] * np.abs(want) * 1.001 + 1e-37 + (6e-8 if self.dtype == "float16" else 0)
        off = np.abs(got[:n] - want[:n]) / bound[:n]
        assert (off <= 1).all(), f"{(off > 1).sum()} of {off.size} off, by {np.nanmax(off)} of the bound"
        return got


CASES = [
    # one row; few; an odd width; a row each in every slot
    (896, (896, 128, 128), 16, 4, [2], [1]),
    (64, (64, 32, 32), 8, 3, [0, 2, 0, 1, -1, 2, 0], [1] * 7),
    (1000, (333,), 32, 9, [5, 3, 3, -1, 8, 0, 1, 2, 3, 4, 5, 6, 7], [1] * 13),
    (4864, (896,), 64, 24, list(range(24)), [1] * 24),
    (8, (1,), 8, 1, [0, 0, -1], [1] * 3),
    (264, (17, 5, 1, 2, 16, 15, 31, 33), 24, 2, [1, 0, 1, 0, 0], [1] * 5),
    (512, (96, 40), 128, 3, [0, 1, 2, 1], [1] * 4),
    # several rows of a sequence: tiles of 16, 32 and 128 rows, with empty sequences
    (896, (896, 128, 128), 16, 8, [3, 3, 1, -1, 7], [13, 0, 5, 9, 21]),
    (128, (130,), 64, 2, [0, 1, 0], [40, 1, 55]),
    (896, (896, 128, 128), 16, 1, [0], [512]),
    (320, (256, 64), 40, 2, [0, 1, -1, 0], [700, 129, 257, 1]),
    (96, (64, 64), 64, 1, [0, 0], [127, 2]),
]


@pytest.mark.parametrize("dtype,wtype", [("float32", BF16), ("float32", "float16"), ("float16", "float16"), (BF16, BF16), (BF16, "float16")])
@pytest.mark.parametrize("inputs,widths,rank,slots,adapters,counts", CASES)
def test_adapters(cuda, dtype, wtype, inputs, widths, rank, slots, adapters, counts):
    Adapted(1, dtype, wtype, inputs, widths, rank, slots, adapters, counts).run().check()


@pytest.mark.parametrize("inputs,widths,rank,slots,adapters,counts", CASES + [(4096, (1024, 40), 32, 3, [0, 2, 1, 0], [1] * 4)])
def test_float16_rows_beside_bfloat16_adapters(cuda, inputs, widths, rank, slots, adapters, counts):
    Adapted(27, "float16", BF16, inputs, widths, rank, slots, adapters, counts).run().check()


@pytest.mark.parametrize("dtype,wtype", [("float16", BF16), (BF16, "float16")])
@pytest.mark.parametrize("inputs,counts", [(256, [1] * 6), (4096, [1] * 6), (256, [90, 3, 200, 1, 0, 17])])
def test_rows_and_adapters_of_different_16_bit_types(cuda, dtype, wtype, inputs, counts):
    """Adapters of ranks of their own with NaN behind them, and rows with an infinity and a NaN."""
    case = Adapted(28, dtype, wtype, inputs, (1000, 28), 64, 6, [0, 1, 2, 3, 4, 5], counts, ranks=[64, 1, 0, 13, 33, 16])
    kept = case.a.copy(), case.b.copy(), case.x.copy()
    for s, r in enumerate(case.ranks):
        for t in range(2):
            case.a[s, t * 64 + r: (t + 1) * 64] = np.nan
        case.b[s, :, r:] = np.nan
    bad = [case.row_start[0], case.row_start[3]]
    case.x[bad[0], 3], case.x[bad[1], inputs - 1] = np.inf, np.nan
    got = decode(case.run().d_out.numpy(), dtype)
    assert not np.isfinite(got[bad]).any() and np.isnan(got[bad[1]]).all()
    case.a, case.b, case.x = kept
    case.x[bad] = case.base[bad] = got[bad] = 0
    case.check(got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts", [[1] * 6, [90, 3, 200, 1, 0, 17]])
def test_adapters_of_ranks_of_their_own(cuda, dtype, counts):
    wtype = "float16" if dtype == "float16" else BF16
    case = Adapted(2, dtype, wtype, 256, (100, 28), 64, 6, [0, 1, 2, 3, 4, 5], counts, ranks=[64, 1, 0, 13, 33, 16])
    for s, r in enumerate(case.ranks):                                   # what lies past an adapter's rank is not read
        for t in range(2):
            case.a[s, t * 64 + r: (t + 1) * 64] = np.nan
        case.b[s, :, r:] = np.nan
    kept = case.a.copy(), case.b.copy()
    case.run()
    case.a, case.b = (np.nan_to_num(v) for v in kept)
    case.check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts", [[1] * 5, [60, 2, 300, 7, 4]])
@pytest.mark.parametrize("stride,skip", [(0, 0), (9, 0), (8, 8), (1, 1)])
def test_strides_alignments_and_outputs_in_place(cuda, dtype, counts, stride, skip):
    case = Adapted(3, dtype, "float16" if dtype == "float16" else BF16, 72, (40, 21), 16, 2, [1, -1, 0, 1, 0], counts)
    x, _ = strided(case.x, dtype, 72 + stride, skip)
    base, _ = strided(case.base, dtype, 61 + stride, skip)
    out, room = strided(np.full_like(case.base, 55), dtype, 61 + 2 * stride, skip)
    case.run(x, base, out)
    rows, line = case.base.shape

    def seen(array, step):
        flat = decode(array.numpy(), dtype).ravel()
        inside = np.arange(rows)[:, None] * step + skip + np.arange(line)
        rest = np.delete(flat, inside.ravel())
        assert (rest == 77).all()                                        # nothing is written beside the rows
        return flat[inside]

    first = case.check(seen(room, 61 + 2 * stride))
    base, room = strided(case.base, dtype, 61 + stride, skip)
    case.run(x, base, base)                                              # out is base
    assert (seen(room, 61 + stride) == first).all()


def test_without_base_scales_or_ranks(cuda):
    case = Adapted(4, "float32", BF16, 128, (48,), 8, 2, [0, -1, 1], [2, 3, 1], scales=False, base=False)
    got = case.run().check()
    assert (got[2:5] == 0).all()


def test_rows_behind_the_last_sequence_stay_as_they_were(cuda):
    case = Adapted(5, "float32", BF16, 128, (48,), 8, 2, [0, 1], [2, 3], tail=4)
    got = case.run().check()
    assert (got[5:] == 55).all()


@pytest.mark.parametrize("counts", [[1] * 3, [150, 20, 3]])
@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_nan_stay_in_their_rows(cuda, dtype, counts):
    case = Adapted(6, dtype, "float16" if dtype == "float16" else BF16, 64, (32,), 16, 1, [0, 0, -1], counts)
    bad = [0, counts[0]]
    case.x[bad[0], 3], case.x[bad[1], 5] = np.inf, np.nan
    got = decode(case.run().d_out.numpy(), dtype)
    assert not np.isfinite(got[bad]).any() and np.isnan(got[bad[1]]).all()
    case.x[bad] = 0
    case.base[bad] = got[bad] = 0
    case.check(got)


def test_an_infinity_is_one_in_float32(cuda):
    case = Adapted(7, "float32", BF16, 64, (32,), 8, 1, [0], [1], base=False, scales=False)
    case.a[...], case.b[...] = 1, 1
    case.x[0, 5] = np.inf
    assert (case.run().d_out.numpy() == np.inf).all()
    case.x[0] = 0
    case.x[0, 7] = 3.4e38                                                # rounds to an infinity in 11 bits
    case.b[..., 1:] = 0
    assert np.allclose(case.run().d_out.numpy(), case.x[0, 7], rtol=2.0 ** -22)


@pytest.mark.parametrize("wtype", [BF16, "float16"])
@pytest.mark.parametrize("rows,inputs,outputs,rank", [(1024, 16384, 64, 8), (8192, 2048, 40, 16), (640, 4096, 96, 64), (1500, 512, 128, 96), (700, 1000, 64, 128),
                                                      (600, 1032, 200, 80)])
@pytest.mark.parametrize("positive", [False, True])
def test_long_float32_prompts_keep_float32_accuracy(cuda, wtype, rows, inputs, outputs, rank, positive):
    """Against the result, where other tests' bounds are of the terms: the matrix unit cuts its sums off at each step, always
    towards nought, which adds up along a chain. A chain of 64 inputs, or of 64 of h, has four steps of full size, each off by
    2^-23 of the sum at most: 2^-21 of h, and as much of the outputs. Up to 32 chains and 8 CTAs' sums are added in float32: 40
    roundings of 2^-25 in the mean, as independent ones 2^-22; the parts that the operands go in, the scale and the output less than 2^-23."""
    case = Adapted(26, "float32", wtype, inputs, (outputs,), rank, 1, [0], [rows], scales=False, base=False)
    if positive:
        case.x, case.a, case.b = np.abs(case.x), np.abs(case.a), np.abs(case.b)
    got = case.run().check()
    want, _ = ref.lora(case.x, case.a, case.b, case.widths, rank, case.adapters, case.row_start)
    off = float(np.sqrt(np.mean((got - want) ** 2) / np.mean(want ** 2)))
    assert off <= 2.0 ** -20 + 2.0 ** -22 + 2.0 ** -23


@pytest.mark.parametrize("wtype", [BF16, "float16"])
@pytest.mark.parametrize("count", [8, 300])
def test_the_largest_numbers_of_float32_rows(cuda, wtype, count):
    """What rounds to an infinity in 16 bits, and an infinity."""
    case = Adapted(16, "float32", wtype, 64, (32,), 8, 1, [0], [count], base=False, scales=False)
    case.a[...], case.b[...] = 1, 0
    case.b[..., 0] = 1
    case.x[1], case.x[2], case.x[5, 9] = 0, 0, np.inf
    case.x[1, 7], case.x[2, 40] = 3.4e38, -3.39e38
    got = case.run().d_out.numpy()
    assert np.allclose(got[1], 3.4e38, rtol=2.0 ** -22) and np.allclose(got[2], -3.39e38, rtol=2.0 ** -22)
    assert np.isnan(got[5]).all()                                        # every h is infinite, and seven of them are multiplied by 0
    case.x[5] = got[5] = 0
    case.check(got)


def test_adapters_outside_the_slots_are_none_and_recorded(cuda):
    error = error_word()
    case = Adapted(8, "float32", BF16, 64, (32,), 8, 3, [1, 7, -5, 3, 2], [1, 2, 1, 1, 4]).run(error=error)
    case.check()
    assert error.numpy()[0] == 1


def test_row_for_each_sequence_and_many_sequences(cuda):
    rng = np.random.default_rng(9)
    for seqs, slots in ((1, 1), (2, 50), (333, 7), (1025, 2000), (8192, 64)):
        Adapted(10, "float32", BF16, 16, (24,), 8, slots, rng.integers(-1, slots, seqs), [1] * seqs).run(by_row=True).check()


@pytest.mark.parametrize("seed", range(6))
def test_ragged_batches(cuda, seed):
    rng = np.random.default_rng(100 + seed)
    seqs, slots = int(rng.integers(1, 40)), int(rng.integers(1, 12))
    counts = [int(c) for c in np.where(rng.random(seqs) < 0.2, 0, np.exp(rng.uniform(0, 5.5, seqs)))]
    Adapted(seed, TYPES[seed % 3], "float16" if seed % 3 == 1 else BF16, 8 * int(rng.integers(1, 60)),
            tuple(int(w) for w in rng.integers(1, 200, int(rng.integers(1, 5)))), 8 * int(rng.integers(1, 9)), slots,
            rng.integers(-1, slots, seqs), counts).run().check()


def test_a_row_start_that_does_not_ascend_stays_in_bounds(cuda):
    case = Adapted(11, "float32", BF16, 64, (32,), 8, 2, [0, 1, 0, 1], [3, 3, 3, 3])
    case.row_start = np.array([5, 2, 400, -7, 12], np.int32)
    case.run().d_out.numpy()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inputs,rows,row_start", [(64, 12, [5, 2, 400, -7, 12]), (4096, 12, [12, -3, 12, 0, 12]), (64, 700, [650, 0, 700, -7, 9000]),
                                                   (64, 700, [0, 700, 0, 700, 0]), (64, 700, [700] * 5)])
def test_a_row_start_that_does_not_ascend_writes_its_rows_alone(cuda, dtype, inputs, rows, row_start):
    """Items of eight rows and of 128: what lies before, between and behind the outputs' rows stays as it was."""
    case = Adapted(29, dtype, "float16" if dtype == "float16" else BF16, inputs, (320, 16), 32, 2, [0, 1, 0, 1], [rows // 4] * 4)
    case.row_start = np.array(row_start, np.int32)
    stride, skip = 336 + 24, 256
    out, room = strided(np.full((rows, 336), 77), dtype, stride, skip)
    _, behind = strided(np.full((rows, 336), 77), dtype, stride, skip)
    case.run(out=out)
    flat = decode(room.numpy(), dtype)
    flat[skip + np.arange(rows)[:, None] * stride + np.arange(336)] = 77
    assert (flat == 77).all() and (decode(behind.numpy(), dtype) == 77).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,inputs,rank", [([1] * 9, 256, 16), ([1] * 9, 4096, 32), ([300], 256, 16), ([128, 1, 256], 256, 16)])
def test_rows_of_a_plan_that_are_none_of_the_call(cuda, dtype, counts, inputs, rank):
    """They are neither read nor written, wherever they lie in an item: a plan's last words are its rows."""
    case = Adapted(23, dtype, "float16" if dtype == "float16" else BF16, inputs, (256, 64), rank, 3, [i % 3 for i in range(len(counts))], counts)
    case.run()
    rows = case.batch.rows
    plan = case.plan.numpy().copy()
    order = plan[plan.size - 4 * rows:].view(np.int32)
    at = [0, rows // 2, rows - 1]
    none = order[at].copy()
    order[at] = -1, rows, -2 ** 31
    assert len(set(none.tolist())) == 3 and ((none >= 0) & (none < rows)).all()
    case.plan.upload(plan)
    case.d_out.upload(encode(np.full((rows, 320), 55, np.float32), dtype))
    serving.lora_project(case.layout, case.batch, case.d_out, case.d_x, case.d_a, case.d_b, case.plan, base=case.d_base, scales=case.d_scales)
    got = decode(case.d_out.numpy(), dtype)
    assert (got[none] == 55).all()
    got[none] = ref.lora(case.x, case.a, case.b, case.widths, rank, case.adapters, case.row_start, case.base, None, case.scales)[0][none]
    case.check(got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,other", [(([1] * 9, 256), ([1] * 10, 256)), (([1] * 9, 4096), ([2] + [1] * 8, 4096)), (([300, 2], 256), ([300, 3], 256)),
                                         (([300, 212], 256), ([512], 256)), (([128, 128, 256], 256), ([1] * 600, 256)), (([600], 256), None)])
def test_a_plan_of_other_sizes_changes_nothing_and_is_reported(cuda, dtype, batch, other):
    """A plan that lies in a buffer for both, of another batch or of none."""
    wtype = "float16" if dtype == "float16" else BF16
    case = Adapted(24, dtype, wtype, batch[1], (256, 64), 32, 3, [i % 3 for i in range(len(batch[0]))], batch[0]).run()
    case.check()
    room = DeviceArray.zeros((1 << 16,), np.uint8)
    if other:
        stale = Adapted(25, dtype, wtype, other[1], (256, 64), 32, 3, [i % 3 for i in range(len(other[0]))], other[0])
        serving.lora_plan(stale.batch, room, DeviceArray.of(stale.adapters), row_start=DeviceArray.of(stale.row_start))
    runtime.device_faults()
    case.d_out.upload(encode(np.full((case.batch.rows, 320), 55, np.float32), dtype))
    project = lambda plan: serving.lora_project(case.layout, case.batch, case.d_out, case.d_x, case.d_a, case.d_b, plan, base=case.d_base,      # noqa: E731
                                                scales=case.d_scales)
    project(room)
    assert (decode(case.d_out.numpy(), dtype) == 55).all()
    with pytest.raises(runtime.KernelError, match="other rows, sequences or slots"):
        runtime.device_faults()
    project(case.plan)
    case.check()
    runtime.device_faults()


def test_no_rows(cuda):
    case = Adapted(12, "float32", BF16, 64, (32,), 8, 2, [], [])
    assert case.run().d_out.numpy().shape == (0, 32)


def test_a_plan_serves_many_projections_and_streams(cuda):
    """A plan and projections captured into a graph and replayed with other adapters, beside calls on the default stream."""
    torch = pytest.importorskip("torch")
    case = Adapted(13, "float32", BF16, 128, (64, 32), 16, 5, [0, 1, 2], [1, 1, 1])
    case.upload()
    put = lambda v: torch.from_numpy(np.ascontiguousarray(v)).cuda()                                  # noqa: E731
    x, base, a, b = put(case.x), put(case.base), put(case.a).bfloat16(), put(case.b).bfloat16()
    scales, adapters = put(case.scales), put(case.adapters)
    out, plan = torch.empty_like(base), torch.zeros(case.batch.plan_bytes, dtype=torch.uint8, device="cuda")

    def step():
        at = torch.cuda.current_stream().cuda_stream
        serving.lora_plan(case.batch, plan, adapters, stream=at)
        serving.lora_project(case.layout, case.batch, out, x, a, b, plan, base=base, scales=scales, stream=at)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    case.check(out.cpu().numpy())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for ids in ([4, -1, 4], [3, 2, 1]):
        case.adapters = np.array(ids, np.int32)
        adapters.copy_(put(case.adapters))
        graph.replay()
        torch.cuda.synchronize()
        case.check(out.cpu().numpy())


@pytest.mark.parametrize("dtype,wtype", [("float32", BF16), ("float16", "float16"), (BF16, BF16)])
@pytest.mark.parametrize("items", [1, 15, 16, 22, 26, 33, 45, 74, 148, 149])
def test_prompts_of_every_cluster_size(cuda, dtype, wtype, items):
    """Rows of one adapter in so many whole items of 128, and one row more."""
    Adapted(17, dtype, wtype, 136, (64, 72), 80, 1, [0], [128 * (items - 1) + 1]).run().check()


@pytest.mark.parametrize("dtype,wtype", [("float32", BF16), ("float32", "float16"), ("float16", "float16"), ("float16", BF16), (BF16, BF16), (BF16, "float16")])
@pytest.mark.parametrize("rank", [88, 96, 104, 128])
@pytest.mark.parametrize("inputs,widths,counts", [(136, (64, 72), [300, 1, 128]), (520, (200, 16, 33), [129, 700])])
def test_prompts_of_large_ranks(cuda, dtype, wtype, rank, inputs, widths, counts):
    """Three or four blocks of B, one target to a pass or two; float32 rows beside float16 adapters above rank 96 in the general kernel."""
    slots = len(counts)
    Adapted(30, dtype, wtype, inputs, widths, rank, slots, list(range(slots)), counts).run().check()
    Adapted(31, dtype, wtype, inputs, widths, rank, slots, list(range(slots)), counts, ranks=[rank - 7] + [rank - 40] * (slots - 1)).run().check()


@pytest.mark.parametrize("dtype,wtype", [("float32", BF16), (BF16, BF16)])
@pytest.mark.parametrize("seqs", [1, 15, 33, 37, 45, 56, 71, 93, 148, 296, 300])
def test_single_tokens_of_every_cluster_size(cuda, dtype, wtype, seqs):
    Adapted(18, dtype, wtype, 1024, (256, 40), 32, seqs, list(range(seqs)), [1] * seqs).run().check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inputs,widths,rank,counts", [(64, (32, 7), 8, [1] * 4), (4864, (896,), 64, [1] * 4), (256, (160, 33), 32, [90, 3, 200, 1])])
def test_adapters_of_rank_nought_are_none(cuda, dtype, inputs, widths, rank, counts):
    """Whatever they hold and whatever their scale: base as it is, also in place."""
    wtype = "float16" if dtype == "float16" else BF16
    case = Adapted(14, dtype, wtype, inputs, widths, rank, 4, [0, 1, 2, 1], counts, ranks=[rank, 0, -3, rank])
    case.a[1:3] = case.b[1:3] = np.nan
    case.scales[1:3] = np.inf, np.nan
    got = decode(case.run().d_out.numpy(), dtype)
    base = device(case.base, dtype)
    in_place = decode(case.run(base=base, out=base).d_out.numpy(), dtype)
    for i in (1, 2, 3):
        at = slice(case.row_start[i], case.row_start[i + 1])
        assert (got[at] == case.base[at]).all() and (in_place[at] == case.base[at]).all()
    case.a[1:3] = case.b[1:3] = 0
    case.scales[1:3] = 1
    case.check(got)
    case.check(in_place)


def test_calls_on_two_streams_at_once(cuda):
    """Plans and projections of different kernels, each stream with a plan of its own."""
    torch = pytest.importorskip("torch")
    cases = [Adapted(19, "float32", BF16, 512, (256, 64), 32, 3, [0, 2, 1], [300, 5, 200]), Adapted(20, BF16, BF16, 1024, (512,), 64, 40, list(range(40)), [1] * 40),
             Adapted(21, "float16", "float16", 256, (640,), 16, 2, [1, 0], [700, 129]), Adapted(22, "float32", "float16", 64, (48,), 8, 4, [3, -1, 0], [1, 1, 1])]
    streams = [torch.cuda.Stream() for _ in cases]
    for case in cases:
        case.run()                                                       # its arrays
    torch.cuda.synchronize()
    for case in cases:
        case.d_out.upload(np.zeros_like(case.d_out.numpy()))
    for _ in range(20):
        for case, stream in zip(cases, streams):
            serving.lora_plan(case.batch, case.plan, case.d_adapters, row_start=case.d_start, stream=stream.cuda_stream)
            serving.lora_project(case.layout, case.batch, case.d_out, case.d_x, case.d_a, case.d_b, case.plan, base=case.d_base, scales=case.d_scales,
                                 stream=stream.cuda_stream)
    torch.cuda.synchronize()
    for case in cases:
        case.check()


# -- beams -----------------------------------------------------------------------------------------------------


class Beams:
    def __init__(self, logits, scores, beams, dtype="float32", end=-1, finished=None, norms=None, stride=None, skip=0):
        rows, vocab = logits.shape
        self.host = rounded(logits, dtype)
        self.logits, self.room = strided(self.host, dtype, stride or vocab, skip)
        self.scores, self.beams, self.end = np.asarray(scores, np.float32), beams, end
        self.finished = None if finished is None else np.asarray(finished, np.int32)
        self.norms = None if norms is None else np.asarray(norms, np.float32)
        self.scratch = DeviceArray.zeros((serving.beam_select_scratch_bytes(rows, vocab, beams),), np.uint8)

    def run(self, error=None, scratch=None):
        rows = self.host.shape[0]
        opt = lambda v: None if v is None else DeviceArray.of(v)                                     # noqa: E731
        out = [DeviceArray.of(np.full(rows, 99, t)) for t in (np.int32, np.int64, np.float32, np.int32, np.int32, np.int32)]
        serving.beam_select(*out[:3], self.logits, DeviceArray.of(self.scores), scratch or self.scratch, beams=self.beams, end=self.end,
                            finished=opt(self.finished), new_finished=out[3], grow=out[4], history=out[5], norms=opt(self.norms), error=error)
        self.got = [v.numpy() for v in out]
        return self

    def check(self):
        rows, width = self.host.shape[0], self.beams
        for g, found in enumerate(ref.beams(self.host, self.scores, width, self.end, self.finished, self.norms)):
            at = slice(g * width, (g + 1) * width)
            got = list(zip(*(v[at].tolist() for v in self.got)))
            want = ref.beam_outputs(found, width, self.end)
            for i, (have, expected) in enumerate(zip(got, want)):
                if have[0] < 0 or expected[0] < 0:
                    assert have == expected, (g, i)
                    continue
                close = 4e-6 + 2.0 ** -22 * abs(expected[2])
                if have[:2] != expected[:2]:                             # allowed for totals that lie this close together alone
                    scale = 1.0 if self.norms is None else float(self.norms[at].min())
                    order = {(c[1], c[2]): c[0] for c in found}
                    assert abs(order[have[:2]] - found[i][0]) <= close / scale, (g, i, have, expected)
                    expected = next(e for e in ref.beam_outputs([c for c in found if (c[1], c[2]) == have[:2]], 1, self.end))
                assert have[3:] == expected[3:], (g, i)
                assert abs(have[2] - expected[2]) <= close, (g, i)
            taken = [h[:2] for h in got if h[0] >= 0]
            assert len(set(taken)) == len(taken)
        assert rows == len(self.got[0])
        return self


def language(rng, rows, vocab):
    logits = rng.standard_normal((rows, vocab)).astype(np.float32) * 2
    for r in range(rows):
        logits[r, rng.integers(0, vocab, 8)] += rng.uniform(0, 12, 8)
    return logits


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups,beams,vocab", [(1, 1, 1), (1, 4, 2), (3, 3, 32), (1, 4, 151936), (2, 32, 40000), (5, 8, 50257), (40, 2, 1001),
                                                (1, 5, 300001)])
def test_beams(cuda, dtype, groups, beams, vocab):
    rng = np.random.default_rng(vocab + beams)
    rows = groups * beams
    Beams(language(rng, rows, vocab), rng.standard_normal(rows) * 2 - 9, beams, dtype).run().check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [7, 5000, 70001])
def test_beams_that_have_finished_or_are_not_there(cuda, dtype, vocab):
    rng = np.random.default_rng(vocab)
    groups, beams = 6, 5
    rows = groups * beams
    scores = rng.standard_normal(rows) * 2 - 5
    scores[rng.random(rows) < 0.3] = -np.inf
    scores[:beams] = -np.inf                                             # a request without beams
    finished = (rng.random(rows) < 0.3).astype(np.int32) * 3
    finished[beams: 2 * beams] = 1                                       # and one of which all have finished
    logits = language(rng, rows, vocab)
    logits[2 * beams: 3 * beams, 3] += 20                                # one whose beams end now
    case = Beams(logits, scores, beams, dtype, end=3, finished=finished, norms=rng.uniform(1, 4, rows)).run().check()
    assert (case.got[0][:beams] == -1).all() and (case.got[1][:beams] == 3).all() and (case.got[5][beams: 2 * beams] == -1).all()


def test_the_first_step_has_one_beam(cuda):
    rng = np.random.default_rng(0)
    logits = language(rng, 8, 3000)
    scores = np.where(np.arange(8) % 4 == 0, 0.0, -np.inf)
    case = Beams(logits, scores, 4).run().check()
    assert (case.got[0] == np.arange(8) // 4 * 4).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [64, 9000, 151936])
def test_equal_totals_go_to_the_lower_beam_and_token(cuda, dtype, vocab):
    logits = np.zeros((6, vocab))
    case = Beams(logits, [-1, -1, -1, -2, -1, -1], 3, dtype).run()
    assert case.got[0].tolist() == [0, 0, 0, 4, 4, 4] and case.got[1].tolist() == [0, 1, 2] * 2
    logits[:, [vocab - 1, vocab // 2]] = 1.0
    case = Beams(logits, np.full(6, -1.0), 6, dtype).run()
    assert case.got[0].tolist() == [0, 0, 1, 1, 2, 2] and case.got[1].tolist() == [vocab // 2, vocab - 1] * 3


def test_forbidden_tokens_are_not_chosen(cuda):
    logits = np.full((8, 500), -np.inf)
    logits[0, [7, 400]] = 1.0, 2.0
    logits[2, 9] = -50.0
    case = Beams(logits, np.zeros(8), 4).run().check()
    assert case.got[0].tolist() == [2, 0, 0, -1] + [-1] * 4 and case.got[1][:3].tolist() == [9, 400, 7]
    assert np.isneginf(case.got[2][3:]).all() and (case.got[3][3:] == 1).all() and (case.got[4][3:] == 0).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("vocab", [50, 60000])
def test_a_beam_with_a_nan_or_infinity_has_no_candidates_and_is_recorded(cuda, bad, vocab):
    rng = np.random.default_rng(3)
    logits = language(rng, 12, vocab)
    logits[5, vocab // 3] = bad
    error = error_word()
    case = Beams(logits, rng.standard_normal(12), 4).run(error).check()
    assert error.numpy()[0] == 5 and 5 not in case.got[0]
    scores = rng.standard_normal(12)
    scores[9] = np.nan
    error = error_word()
    case = Beams(language(rng, 12, vocab), scores, 4, end=2, finished=(np.arange(12) == 10)).run(error).check()
    assert error.numpy()[0] == 9 and 9 not in case.got[0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stride,skip", [(5001, 0), (5003, 1), (5008, 4), (6000, 3)])
def test_logits_at_strides_and_alignments(cuda, dtype, stride, skip):
    rng = np.random.default_rng(stride)
    Beams(language(rng, 6, 5001), rng.standard_normal(6), 3, dtype, stride=stride, skip=skip).run().check()


def test_many_requests_in_several_launches(cuda):
    rng = np.random.default_rng(5)
    Beams(language(rng, 3 * 1400, 40), rng.standard_normal(3 * 1400), 3).run().check()


def test_a_beam_scratch_serves_smaller_calls_and_is_left_as_the_next_needs_it(cuda):
    rng = np.random.default_rng(6)
    scratch = DeviceArray.zeros((serving.beam_select_scratch_bytes(96, 60000, 16),), np.uint8)
    for rows, vocab, beams in ((96, 60000, 16), (4, 60000, 4), (90, 59999, 9), (1, 17, 1), (96, 60000, 16)):
        Beams(language(rng, rows, vocab), rng.standard_normal(rows), beams).run(scratch=scratch).check()


@pytest.mark.parametrize("rows,beams,vocab,smaller", [(4, 4, 132000, 108000), (8, 8, 264000, 234000), (32, 32, 66000, 62000)])
def test_a_beam_scratch_serves_smaller_vocabularies(cuda, rows, beams, vocab, smaller):
    """Also where those are cut into more segments."""
    rng = np.random.default_rng(7)
    scratch = DeviceArray.zeros((serving.beam_select_scratch_bytes(rows, vocab, beams),), np.uint8)
    for n in (vocab, smaller, vocab):
        Beams(language(rng, rows, n), rng.standard_normal(rows), beams).run(scratch=scratch).check()


def test_a_captured_choice_and_its_reordering_follow_their_inputs(cuda):
    """A step captured into a graph, replayed with other logits, scores and states: what the calls outside a graph give."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(15)
    groups, beams, vocab = 3, 4, 20011
    rows = groups * beams
    put = lambda v: torch.from_numpy(np.ascontiguousarray(v)).cuda()                                  # noqa: E731
    logits, scores, states = put(language(rng, rows, vocab)), put(np.zeros(rows, np.float32)), put(rng.standard_normal((rows, 9)).astype(np.float32))
    scratch = torch.zeros(serving.beam_select_scratch_bytes(rows, vocab, beams), dtype=torch.uint8, device="cuda")
    parent, tokens = (torch.empty(rows, dtype=t, device="cuda") for t in (torch.int32, torch.int64))
    totals, moved = torch.empty(rows, device="cuda"), torch.empty_like(states)

    def step():
        at = torch.cuda.current_stream().cuda_stream
        serving.beam_select(parent, tokens, totals, logits, scores, scratch, beams=beams, stream=at)
        serving.beam_reorder(moved, states, parent, stream=at)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for live in (rows, 5, 1):
        case = Beams(language(rng, rows, vocab), np.where(np.arange(rows) < live, rng.standard_normal(rows) - 4, -np.inf), beams).run().check()
        logits.copy_(put(case.host))
        scores.copy_(put(case.scores))
        states.copy_(put(rng.standard_normal((rows, 9)).astype(np.float32)))
        before = moved.cpu().numpy()
        graph.replay()
        torch.cuda.synchronize()
        for have, want in zip((parent, tokens, totals), case.got):
            assert (have.cpu().numpy() == want).all()
        was, now = states.cpu().numpy(), moved.cpu().numpy()
        for i, p in enumerate(case.got[0]):
            assert (now[i] == (was[p] if p >= 0 else before[i])).all()


# -- states ----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["float32", "float16", "int32", "int64", "uint8"])
@pytest.mark.parametrize("rows,planes,capacity,line", [(1, 1, 1, 1), (4, 3, 17, 5), (8, 6, 64, 64), (3, 2, 1000, 33), (5, 1, 4096, 1), (2, 2, 0, 4)])
@pytest.mark.parametrize("mode", ["whole", "lengths", "append", "grow"])
def test_states(cuda, dtype, rows, planes, capacity, line, mode):
    rng = np.random.default_rng(rows * capacity + line)
    old, new = ((rng.standard_normal((rows, planes, capacity, line)) * 100).astype(dtype) for _ in range(2))
    parent = rng.integers(0, rows, rows).astype(np.int32)
    if rows > 2:
        parent[1], parent[2] = -1, rows
    lengths = rng.integers(0, capacity + 1, rows).astype(np.int32)
    lengths[-1] = capacity
    lengths[0] = 0
    append = (rng.standard_normal((rows, planes, line)) * 100).astype(dtype)
    grow = rng.integers(0, 2, rows).astype(np.int32)
    give = {"whole": {}, "lengths": {"lengths": lengths}, "append": {"lengths": lengths, "append": append},
            "grow": {"lengths": lengths, "append": append, "grow": grow}}[mode]
    want, after = ref.reorder(new, old, parent, **give)
    d_new, d_after = DeviceArray.of(new), DeviceArray.of(np.full(rows, 9, np.int32))
    more = {} if mode == "whole" else {"new_lengths": d_after}
    serving.beam_reorder(d_new, DeviceArray.of(old), DeviceArray.of(parent), **{k: DeviceArray.of(v) for k, v in give.items()}, **more)
    assert (d_new.numpy() == want).all()
    if more:
        assert (d_after.numpy() == after).all()


@pytest.mark.parametrize("skip,stride", [(0, 0), (1, 3), (2, 4), (4, 8)])
def test_states_at_strides_and_alignments(cuda, skip, stride):
    rng = np.random.default_rng(skip)
    rows, planes, capacity, line = 4, 2, 12, 6
    old, new = (rng.standard_normal((rows, planes, capacity, line)).astype(np.float16) for _ in range(2))
    size, parent = planes * capacity * line, np.array([2, 2, 0, 3], np.int32)
    lengths = np.array([12, 1, 7, 5], np.int32)

    def room(states):
        flat = np.full(skip + rows * (size + stride), 7, np.float16)
        for i in range(rows):
            flat[skip + i * (size + stride):][:size] = states[i].ravel()
        array = DeviceArray.of(flat)
        return View(array, states.shape, (size + stride, capacity * line, line, 1), skip), array

    (d_new, buffer), (d_old, _) = room(new), room(old)
    serving.beam_reorder(d_new, d_old, DeviceArray.of(parent), lengths=DeviceArray.of(lengths))
    want, _ = ref.reorder(new, old, parent, lengths)
    _, expected = room(want)
    assert (buffer.numpy() == expected.numpy()).all()


def test_lengths_past_the_capacity_are_cut(cuda):
    old, new = np.arange(24, dtype=np.int64).reshape(3, 8), np.zeros((3, 8), np.int64)
    d_new, after = DeviceArray.of(new), DeviceArray.zeros((3,), np.int32)
    serving.beam_reorder(d_new, DeviceArray.of(old), DeviceArray.of(np.array([1, 0, 2], np.int32)), lengths=DeviceArray.of(np.array([99, -4, 8], np.int32)),
                         append=DeviceArray.of(np.array([100, 101, 102], np.int64)), new_lengths=after)
    assert after.numpy().tolist() == [1, 8, 8]
    assert d_new.numpy().tolist() == [[100] + [0] * 7, old[0].tolist(), old[2].tolist()]


def test_states_past_32_bits(cuda):
    """Rows of more than 2^31 bytes, more than 2^32 bytes apart."""
    rows, capacity, size = 3, 3 << 20, 3 << 30
    old, new = (DeviceArray((rows, 1, capacity, 1024), np.uint8) for _ in range(2))
    lib = runtime.library()
    line = np.arange(4096, dtype=np.int64).astype(np.uint8)
    runtime.check(lib.nc_copy_to_device(ctypes.c_void_p(old.data_ptr() + 3 * size - 4096), line.ctypes.data, 4096))
    serving.beam_reorder(new, old, DeviceArray.of(np.array([-1, 2, -1], np.int32)))
    got = np.zeros(4096, np.uint8)
    runtime.check(lib.nc_copy_to_host(got.ctypes.data, ctypes.c_void_p(new.data_ptr() + 2 * size - 4096), 4096))
    assert (got == line).all()


def test_no_wait_has_run_out(cuda):
    """After all of the above: the kernels' waits end because what they wait for comes."""
    runtime.check(runtime.library().nc_device_faults())
