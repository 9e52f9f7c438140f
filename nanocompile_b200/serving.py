"""Serving operators next to the Qwen2 step: a paged key/value cache held in 4 bits, token log probabilities, beams and adapters.

The reference keeps one sequence's history as float32 arrays (``nanocompile/models/qwen2.py:232-271``) and
picks tokens by ``np.argmax`` (``nanocompile/models/qwen2.py:348-368``). Sampling several continuations of a
prompt, or searching with beams, needs more: histories that share their pages (:func:`kv_pages_update` forks,
reorders, grows, cuts and frees sequences, :func:`kv_pages_compact` packs them), at 5 bits a value
(:func:`kv4_append`, :func:`kv4_attention`, :func:`kv4_read`), and the scores of a step's tokens
(:func:`token_logprobs`). The beams of a batch of requests are chosen on the device (:func:`beam_select`), dense states follow
them (:func:`beam_reorder`), and each request may have a low-rank adapter of its own beside the shared projections
(:func:`lora_plan`, :func:`lora_project`). Each function is one entry point of ``libnc_cuda.so`` (``include/nc_cuda.h``).

Arguments are device arrays: anything with ``data_ptr()``, ``shape``, ``stride()``, ``is_contiguous()`` and ``dtype`` --
this module's :class:`DeviceArray`, a PyTorch tensor -- on the current device. Calls are asynchronous on ``stream`` (a CUDA stream
handle; 0 is the default stream) and allocate nothing; scratch is zeroed once by the caller and must not be used by
two calls at once. A refused call raises :class:`~nanocompile_b200.runtime.InterpreterError`.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from functools import cached_property
from struct import Struct

import numpy as np

from nanocompile_b200.runtime import InterpreterError, check, library

_vp, _i64 = ctypes.c_void_p, ctypes.c_int64
_SIZES = {"bfloat16": np.uint16}                        # how NumPy holds what it has no type for


class DeviceArray:
    """A device allocation of one array, in C order. ``dtype``: a NumPy type, or ``"bfloat16"`` (held as uint16)."""

    def __init__(self, shape, dtype):
        self.shape = tuple(int(n) for n in shape)
        self.dtype = dtype if dtype == "bfloat16" else np.dtype(dtype)
        self.host_type = np.dtype(_SIZES.get(str(self.dtype), self.dtype))
        self.nbytes = int(np.prod(self.shape, dtype=np.int64)) * self.host_type.itemsize
        pointer = _vp()
        check(library().nc_device_alloc(max(self.nbytes, 1), ctypes.byref(pointer)))
        self._pointer = pointer.value

    @classmethod
    def of(cls, host: np.ndarray, dtype=None) -> "DeviceArray":
        """A device copy of ``host`` (``dtype="bfloat16"``: of its uint16 bits)."""
        host = np.ascontiguousarray(host)
        out = cls(host.shape, dtype or host.dtype)
        out.upload(host)
        return out

    @classmethod
    def zeros(cls, shape, dtype) -> "DeviceArray":
        out = cls(shape, dtype)
        out.upload(np.zeros(out.shape, out.host_type))
        return out

    def data_ptr(self) -> int:
        return self._pointer

    def stride(self) -> tuple[int, ...]:
        """Elements from one index to the next, by axis."""
        return tuple(int(np.prod(self.shape[axis + 1:], dtype=np.int64)) for axis in range(len(self.shape)))

    def is_contiguous(self) -> bool:
        return True

    def upload(self, host: np.ndarray) -> None:
        host = np.ascontiguousarray(host, self.host_type)
        if host.shape != self.shape:
            raise InterpreterError(f"a host array of shape {host.shape} for a device array of {self.shape}")
        if self.nbytes:
            check(library().nc_copy_to_device(self._pointer, host.ctypes.data, self.nbytes))

    def numpy(self) -> np.ndarray:
        """A host copy, after what the default stream has been given; calls on other streams are to be waited for first."""
        out = np.empty(self.shape, self.host_type)
        if self.nbytes:
            check(library().nc_copy_to_host(out.ctypes.data, self._pointer, self.nbytes))
        return out

    def free(self) -> None:
        if self._pointer:
            library().nc_device_free(self._pointer)
            self._pointer = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def _f32_bits(value: float) -> int:
    return int(np.float32(value).view(np.uint32))


@dataclass(frozen=True)
class KV4Layout:
    """The sizes of a 4-bit paged cache: ``page_size`` positions (a multiple of 16, at most 1024) of ``layers`` layers to a page."""

    heads: int
    kv_heads: int
    head_dim: int
    page_size: int = 64
    layers: int = 1

    def __post_init__(self) -> None:
        if min(self.heads, self.kv_heads, self.layers) <= 0 or self.heads % self.kv_heads:
            raise InterpreterError(f"{self.heads} query heads do not share {self.kv_heads} KV heads evenly")
        if self.head_dim not in (32, 64, 96, 128):
            raise InterpreterError(f"head dimension {self.head_dim}: the 4-bit cache serves 32, 64, 96 and 128")
        if self.page_size <= 0 or self.page_size % 16:
            raise InterpreterError(f"page size {self.page_size}: a multiple of 16 positions")

    @cached_property
    def layer_bytes(self) -> int:
        """A layer's part of a page."""
        return self.kv_heads * self.page_size * self.head_dim * 5 // 4

    @cached_property
    def page_bytes(self) -> int:
        return self.layers * self.layer_bytes

    @cached_property
    def scale_bits(self) -> int:
        """The default score scale, ``head_dim ** -0.5``, as the bits of a float32."""
        return _f32_bits(self.head_dim ** -0.5)

    def pages_for(self, positions: int) -> int:
        return -(-positions // self.page_size)


# The smallest calls take a few microseconds on the device, so the checks before them are kept short: every property of
# an array is asked for once, element types are compared as small numbers, and what is wrong is looked for only
# where something is.
_F32, _F16, _BF16, _I32, _I64, _U64, _U8, _OTHER = range(8)
_NAMES = {"float32": _F32, "float16": _F16, "bfloat16": _BF16, "int32": _I32, "int64": _I64, "uint64": _U64, "uint8": _U8}


class _Kinds(dict):
    """Element types, as arrays give them, to small numbers."""

    def __missing__(self, dtype) -> int:
        kind = self[dtype] = _NAMES.get(_name(dtype), _OTHER)
        return kind


_kind = _Kinds()


def _name(dtype) -> str:
    return str(dtype).removeprefix("torch.")


def _expect(what: str, array, kind: int, shape: tuple) -> int:
    """The address of a contiguous ``array`` of this kind and ``shape``."""
    if array.shape != shape or _kind[array.dtype] != kind or not array.is_contiguous():
        expected = next(name for name, k in _NAMES.items() if k == kind)
        raise InterpreterError(f"{what}: {_name(array.dtype)} {tuple(array.shape)}, expected a contiguous {expected} {shape}")
    return array.data_ptr()


def _rows(what: str, array, heads: int, d: int) -> tuple[int, int, int, int]:
    """Address, rows, row stride and kind of ``[rows, heads * d]`` or ``[rows, heads, d]``; rows may be strided."""
    shape, strides, line, kind = array.shape, array.stride(), heads * d, _kind[array.dtype]
    if len(shape) == 2:
        fits = shape[1] == line and strides[1] == 1
    else:
        fits = len(shape) == 3 and shape[1] == heads and shape[2] == d and strides[2] == 1 and (heads == 1 or strides[1] == d)
    if not fits:
        raise InterpreterError(f"{what}: {tuple(shape)}, expected rows of {heads} contiguous heads of {d}")
    if kind > _BF16:
        raise InterpreterError(f"{what}: element type {_name(array.dtype)}: float32, float16 or bfloat16")
    rows = shape[0]
    return array.data_ptr(), rows, strides[0] if rows > 1 else line, kind


def _rope(rope, d: int) -> tuple[int, int, int]:
    if rope is None:
        return 0, 0, 0
    cos, sin = rope
    shape = cos.shape
    if len(shape) != 2 or shape[1] != d // 2 or sin.shape != shape or _kind[cos.dtype] or _kind[sin.dtype] or not (cos.is_contiguous() and sin.is_contiguous()):
        positions = shape[0] if len(shape) else 0
        _expect("cos", cos, _F32, (positions, d // 2))
        _expect("sin", sin, _F32, (positions, d // 2))
    return cos.data_ptr(), sin.data_ptr(), shape[0]


def _cache(layout: KV4Layout, layer: int, pool, table, lengths, row_start) -> tuple:
    """Addresses of the pool, table, lengths and row starts; sequences, pages, layer offset, table width."""
    shape, held = table.shape, pool.shape
    if not (len(shape) == 2 and len(held) == 2 and held[1] == layout.page_bytes and 0 <= layer < layout.layers
            and _kind[table.dtype] == _kind[lengths.dtype] == _I32 and _kind[pool.dtype] == _U8 and lengths.shape == shape[:1]
            and table.is_contiguous() and lengths.is_contiguous() and pool.is_contiguous()):
        if not 0 <= layer < layout.layers:
            raise InterpreterError(f"layer {layer} of {layout.layers}")
        if len(shape) != 2:
            raise InterpreterError(f"table: {tuple(shape)}, expected [sequences, pages of a sequence]")
        _expect("table", table, _I32, tuple(shape))
        _expect("pool", pool, _U8, (held[0] if len(held) else 0, layout.page_bytes))
        _expect("lengths", lengths, _I32, (shape[0],))
    seqs, width = shape
    return (pool.data_ptr(), table.data_ptr(), lengths.data_ptr(),
            0 if row_start is None else _expect("row_start", row_start, _I32, (seqs + 1,)),
            seqs, held[0], layer * layout.layer_bytes, width)


def _error(array) -> int:
    """The address of an error word, which is written with eight bytes; 0 for none."""
    if array is None:
        return 0
    kind = _kind[array.dtype]
    if kind != _U64 and kind != _I64 or 0 in array.shape:
        raise InterpreterError(f"error: {_name(array.dtype)} {tuple(array.shape)}, expected a word of 64 bits")
    return array.data_ptr()


def _scratch(array) -> tuple[int, int]:
    """Address and bytes of scratch."""
    shape = array.shape
    if len(shape) != 1 or not array.is_contiguous():
        raise InterpreterError(f"scratch: {_name(array.dtype)} {tuple(shape)}, expected contiguous bytes")
    return array.data_ptr(), shape[0]


_entries: dict = {}


def _entry(name: str, pointers: int, sizes: int):
    """The entry point ``name``, taking its p[] and s[] as packed bytes, and their packers."""
    function = ctypes.CFUNCTYPE(ctypes.c_int32, ctypes.c_char_p, ctypes.c_char_p, _vp)((name, library()))
    entry = _entries[name] = (function, Struct(f"{pointers}P").pack, Struct(f"{sizes}q").pack)
    return entry


def _call(name: str, pointers: tuple, sizes: tuple, stream: int) -> None:
    function, pack_p, pack_s = _entries.get(name) or _entry(name, len(pointers), len(sizes))
    status = function(pack_p(*pointers), pack_s(*sizes), stream)
    if status:
        check(status)


def _same_rows(what: str, rows: int, expected: int) -> None:
    if rows != expected:
        raise InterpreterError(f"{what}: {rows} rows, expected {expected}")


def kv4_append(layout: KV4Layout, pool, keys, values, table, lengths, *, row_start=None, rope=None, layer: int = 0,
               error=None, stream: int = 0) -> None:
    """Quantise rows of ``keys`` and ``values`` into the cache (``nc_kv4_append``).

    ``lengths`` are the sequences' lengths after the append: rows ``row_start[i] .. row_start[i + 1] - 1`` become
    the last positions of sequence ``i`` (without ``row_start``, row ``i`` is sequence ``i``'s only one). ``rope``: the
    (cos, sin) tables the keys are rotated by, float32 ``[positions, head_dim / 2]``.
    """
    base, tab, lens, starts, seqs, pages, offset, width = _cache(layout, layer, pool, table, lengths, row_start)
    d, kv = layout.head_dim, layout.kv_heads
    k, rows, k_stride, kind = _rows("keys", keys, kv, d)
    v, v_rows, v_stride, v_kind = _rows("values", values, kv, d)
    _same_rows("values", v_rows, rows)
    if v_kind != kind:
        raise InterpreterError("keys and values of different types")
    cos, sin, positions = _rope(rope, d)
    _call("nc_kv4_append", (base, k, v, tab, lens, starts, cos, sin, _error(error)),
          (rows, seqs, kv, d, layout.page_size, pages, layout.page_bytes, offset, width, k_stride, v_stride, kind, positions),
          stream)


def kv4_read(layout: KV4Layout, keys, values, pool, table, lengths, *, row_start=None, layer: int = 0, error=None,
             stream: int = 0) -> None:
    """The values that the cache holds for rows' positions, to float32 ``[rows, kv_heads * head_dim]`` (``nc_kv4_read``)."""
    base, tab, lens, starts, seqs, pages, offset, width = _cache(layout, layer, pool, table, lengths, row_start)
    d, kv = layout.head_dim, layout.kv_heads
    k, rows, k_stride, kind = _rows("keys", keys, kv, d)
    v, v_rows, v_stride, v_kind = _rows("values", values, kv, d)
    _same_rows("values", v_rows, rows)
    if kind or v_kind or k_stride != kv * d or v_stride != kv * d:
        raise InterpreterError("keys and values: contiguous float32 rows")
    _call("nc_kv4_read", (k, v, base, tab, lens, starts, _error(error)),
          (rows, seqs, kv, d, layout.page_size, pages, layout.page_bytes, offset, width), stream)


def kv4_attention_scratch_bytes(layout: KV4Layout, rows: int, seqs: int, max_length: int, max_rows: int = 1) -> int:
    """Scratch for :func:`kv4_attention` calls of up to these sizes (``rows`` is not needed; a sequence has ``max_rows`` at most)."""
    return int(library().nc_kv4_attention_scratch_bytes(seqs, layout.heads, layout.kv_heads, layout.head_dim, max_rows, max_length))


def kv4_attention(layout: KV4Layout, out, q, pool, table, lengths, scratch, *, max_length: int, row_start=None,
                  max_rows: int = 1, rope=None, layer: int = 0, scale: float | None = None, lse=None, error=None,
                  stream: int = 0) -> None:
    """Attention of the rows ``q`` over the cache, to ``out`` (``nc_kv4_attention``).

    Each row sees its sequence's positions up to its own (rows as in :func:`kv4_append`). ``max_length`` and ``max_rows``
    bound the sequences' lengths and rows; what lies past them is left out. ``scale`` (positive) defaults to
    ``head_dim ** -0.5``. float32 and float16 rows keep float32 accuracy; bfloat16 rows are rounded once to an f16 part.
    ``lse``: float32 ``[rows, heads]`` for the log-sums of the scores.
    """
    base, tab, lens, starts, seqs, pages, offset, width = _cache(layout, layer, pool, table, lengths, row_start)
    d, heads = layout.head_dim, layout.heads
    query, rows, q_stride, kind = _rows("q", q, heads, d)
    to, out_rows, out_stride, out_kind = _rows("out", out, heads, d)
    _same_rows("out", out_rows, rows)
    if out_kind != kind:
        raise InterpreterError("q and out of different types")
    cos, sin, positions = _rope(rope, d)
    bits = layout.scale_bits if scale is None else _f32_bits(scale)
    work, work_bytes = _scratch(scratch)
    _call("nc_kv4_attention",
          (to, query, base, tab, lens, starts, cos, sin, 0 if lse is None else _expect("lse", lse, _F32, (rows, heads)),
           work, _error(error)),
          (rows, seqs, layout.kv_heads, d, layout.page_size, pages, layout.page_bytes, offset, width, heads, q_stride,
           out_stride, kind, positions, bits, max_rows, max_length, work_bytes), stream)


def kv_pages_scratch_bytes(seqs: int, width: int, pages: int) -> int:
    """Scratch for :func:`kv_pages_update` and :func:`kv_pages_compact`."""
    return int(library().nc_kv_pages_scratch_bytes(seqs, width, pages))


def _pages(new_table, table, lengths, pool, status, scratch, page_size: int) -> tuple[tuple, tuple]:
    shape, held = table.shape, pool.shape
    if len(shape) != 2 or len(held) != 2:
        raise InterpreterError(f"table {tuple(shape)} and pool {tuple(held)}: expected [sequences, pages] and [pages, bytes]")
    (seqs, width), (pages, page_bytes) = shape, held
    work, work_bytes = _scratch(scratch)
    return ((_expect("new_table", new_table, _I32, shape), _expect("table", table, _I32, shape),
             _expect("lengths", lengths, _I32, (seqs,)), _expect("status", status, _I64, (4,)),
             _expect("pool", pool, _U8, held), work),
            (seqs, width, pages, page_size, page_bytes, work_bytes))


def kv_pages_update(new_table, new_lengths, table, lengths, pool, status, scratch, *, page_size: int, parent=None,
                    grow=None, stream: int = 0) -> None:
    """Fork, reorder, grow, cut and free a cache's sequences (``nc_kv_pages_update``).

    New sequence ``i`` continues ``parent[i]`` (default: itself; -1: none) at its length plus ``grow[i]`` (default 0).
    ``status`` (int64 ``[4]``): pages missing (then nothing is changed), pages in use, pages copied, highest id in use + 1.
    """
    (new, old, lens, state, base, work), sizes = _pages(new_table, table, lengths, pool, status, scratch, page_size)
    n = (sizes[0],)
    _call("nc_kv_pages_update",
          (new, _expect("new_lengths", new_lengths, _I32, n), old, lens, state, base, work,
           0 if parent is None else _expect("parent", parent, _I32, n),
           0 if grow is None else _expect("grow", grow, _I32, n)), sizes, stream)


def kv_pages_compact(new_table, table, lengths, pool, status, scratch, *, page_size: int, stream: int = 0) -> None:
    """Move the pages in use to the lowest ids (``nc_kv_pages_compact``)."""
    (new, old, lens, state, base, work), sizes = _pages(new_table, table, lengths, pool, status, scratch, page_size)
    _call("nc_kv_pages_compact", (new, 0, old, lens, state, base, work), sizes, stream)


def token_logprobs_scratch_bytes(rows: int, vocab: int, top: int) -> int:
    """Scratch for :func:`token_logprobs` calls of up to ``rows`` rows."""
    return int(library().nc_token_logprobs_scratch_bytes(rows, vocab, top))


def token_logprobs(logits, targets, out, entropy=None, top=None, top_logprobs=None, *, lse=None, scratch=None, error=None,
                   stream: int = 0) -> None:
    """Log probabilities of ``targets`` (int64 ``[rows, n]``) under rows of ``logits``, to ``out`` (``nc_token_logprobs``).

    ``entropy`` and ``lse``: float32 ``[rows]``. ``top`` (int64) and ``top_logprobs`` (float32), both or neither, ``[rows, k]``
    with ``k`` up to 32: the best tokens, in order.
    """
    shape, strides = logits.shape, logits.stride()
    if len(shape) != 2 or strides[1] != 1:
        raise InterpreterError(f"logits: {tuple(shape)}, expected [rows, vocabulary] with contiguous rows")
    rows, vocab = shape
    kind = _kind[logits.dtype]
    if kind > _BF16:
        raise InterpreterError(f"logits: element type {_name(logits.dtype)}: float32, float16 or bfloat16")
    if (top is None) != (top_logprobs is None) or (targets is not None and out is None):
        raise InterpreterError("targets go with out, and top with top_logprobs")
    n = targets.shape[-1] if targets is not None else 0
    k = top.shape[-1] if top is not None else 0
    work, work_bytes = (0, 0) if scratch is None else _scratch(scratch)
    _call("nc_token_logprobs",
          (_expect("out", out, _F32, (rows, n)) if n else 0,
           0 if entropy is None else _expect("entropy", entropy, _F32, (rows,)),
           0 if lse is None else _expect("lse", lse, _F32, (rows,)),
           _expect("top", top, _I64, (rows, k)) if k else 0,
           _expect("top_logprobs", top_logprobs, _F32, (rows, k)) if k else 0,
           logits.data_ptr(), _expect("targets", targets, _I64, (rows, n)) if n else 0,
           work, _error(error)),
          (rows, vocab, strides[0] if rows > 1 else vocab, kind, n, k, work_bytes), stream)


@dataclass(frozen=True)
class LoraBatch:
    """The sizes of a batch: ``rows`` of ``seqs`` sequences (8192 at most), whose adapters are among ``slots``."""

    rows: int
    seqs: int
    slots: int

    def __post_init__(self) -> None:
        if min(self.rows, self.seqs) < 0 or self.slots <= 0 or self.seqs > 8192:
            raise InterpreterError(f"{self.rows} rows of {self.seqs} sequences (8192 at most), {self.slots} adapters")

    @cached_property
    def plan_bytes(self) -> int:
        """The bytes of a plan (at a 16-byte boundary) for :func:`lora_plan`."""
        return int(library().nc_lora_plan_bytes(self.rows, self.seqs, self.slots))


@dataclass(frozen=True)
class LoraLayout:
    """Adapters of up to ``rank`` (a multiple of 8, at most 128) on projections of ``inputs`` (a multiple of 8) that share their rows:
    ``widths`` are their outputs (eight projections at most)."""

    inputs: int
    widths: tuple[int, ...]
    rank: int

    def __post_init__(self) -> None:
        object.__setattr__(self, "widths", tuple(int(w) for w in self.widths))
        if self.inputs <= 0 or self.inputs % 8 or not 0 < self.rank <= 128 or self.rank % 8:
            raise InterpreterError(f"{self.inputs} inputs, rank {self.rank}: multiples of 8, the rank at most 128")
        if not 0 < len(self.widths) <= 8 or min(self.widths) <= 0:
            raise InterpreterError(f"outputs {self.widths}: of one to eight projections")

    @cached_property
    def outputs(self) -> int:
        return sum(self.widths)

    def a_shape(self, slots: int) -> tuple[int, int, int]:
        """The adapters' first factors: ``[slots, projections * rank, inputs]``."""
        return slots, len(self.widths) * self.rank, self.inputs

    def b_shape(self, slots: int) -> tuple[int, int, int]:
        """Their second factors: ``[slots, outputs, rank]``."""
        return slots, self.outputs, self.rank


def lora_plan(batch: LoraBatch, plan, adapters, *, row_start=None, error=None, stream: int = 0) -> None:
    """Group the rows of a batch by adapter, to ``plan`` (uint8), for every :func:`lora_project` of the batch (``nc_lora_plan``).

    ``adapters``: int32 ``[seqs]``, each sequence's slot, -1 for none. ``row_start``: int32 ``[seqs + 1]`` (default: one row each).
    """
    work, work_bytes = _scratch(plan)
    seqs = batch.seqs
    _call("nc_lora_plan", (work, _expect("adapters", adapters, _I32, (seqs,)),
                           0 if row_start is None else _expect("row_start", row_start, _I32, (seqs + 1,)), _error(error)),
          (batch.rows, seqs, batch.slots, work_bytes), stream)


def _lora_rows(what: str, array, rows: int, line: int) -> tuple[int, int, int]:
    """Address, row stride and kind of ``[rows, line]`` with contiguous rows."""
    shape, strides, kind = array.shape, array.stride(), _kind[array.dtype]
    if len(shape) != 2 or shape[0] != rows or shape[1] != line or strides[1] != 1 and line > 1:
        raise InterpreterError(f"{what}: {tuple(shape)}, expected {rows} contiguous rows of {line}")
    if kind > _BF16:
        raise InterpreterError(f"{what}: element type {_name(array.dtype)}: float32, float16 or bfloat16")
    return array.data_ptr(), strides[0] if rows > 1 else line, kind


def lora_project(layout: LoraLayout, batch: LoraBatch, out, x, a, b, plan, *, base=None, ranks=None, scales=None,
                 stream: int = 0) -> None:
    """Add the adapters' shares to the outputs of projections of ``x`` (``nc_lora_project``).

    ``out`` = ``base`` (default: nought; may be ``out`` itself, at its stride) + ``scales`` * B (A x), each row with its sequence's adapter.
    ``a`` and ``b``: float16 or bfloat16, as :meth:`LoraLayout.a_shape` and ``b_shape`` say. ``ranks`` (int32 ``[slots]``): the adapters' own
    ranks, where lower; ``scales``: float32 ``[slots]``. float32 rows keep float32 accuracy (few rows beside float16 adapters: to 2^-39 of
    the row's largest value, where that is coarser). With a plan of another batch's sizes
    ``out`` stays as it was, and ``runtime.device_faults`` raises.
    """
    rows, slots = batch.rows, batch.slots
    to, out_stride, kind = _lora_rows("out", out, rows, layout.outputs)
    source, x_stride, x_kind = _lora_rows("x", x, rows, layout.inputs)
    was, base_stride, base_kind = (0, 0, kind) if base is None else _lora_rows("base", base, rows, layout.outputs)
    if x_kind != kind or base_kind != kind:
        raise InterpreterError("x, base and out of different types")
    weights = _kind[a.dtype]
    if weights != _F16 and weights != _BF16:
        raise InterpreterError(f"a: element type {_name(a.dtype)}: float16 or bfloat16")
    work, work_bytes = _scratch(plan)
    widths = layout.widths + (0,) * (8 - len(layout.widths))
    _call("nc_lora_project",
          (to, source, was, _expect("a", a, weights, layout.a_shape(slots)), _expect("b", b, weights, layout.b_shape(slots)), work,
           0 if ranks is None else _expect("ranks", ranks, _I32, (slots,)),
           0 if scales is None else _expect("scales", scales, _F32, (slots,))),
          (rows, batch.seqs, slots, layout.inputs, layout.rank, len(layout.widths), kind, weights, work_bytes, x_stride, base_stride,
           out_stride, *widths), stream)


def beam_select_scratch_bytes(rows: int, vocab: int, beams: int) -> int:
    """Scratch for :func:`beam_select` calls of up to ``rows`` rows of ``vocab`` logits and ``beams`` beams."""
    return int(library().nc_beam_select_scratch_bytes(rows, vocab, beams))


def beam_select(parent, tokens, new_scores, logits, scores, scratch, *, beams: int, end: int = -1, finished=None, new_finished=None,
                grow=None, history=None, norms=None, error=None, stream: int = 0) -> None:
    """The ``beams`` (32 at most) best continuations of each request's beams (``nc_beam_select``).

    Rows ``g * beams ..`` of ``logits`` and ``scores`` (float32 ``[rows]``, -inf: no beam) are request ``g``'s. A beam for which
    ``finished`` (int32) is not 0 goes on as itself, with the token ``end``. Totals are compared over ``norms`` (float32, positive),
    where given. Out: ``parent`` (int32: rows, -1 for none), ``tokens`` (int64), ``new_scores``, and where wanted ``new_finished``, ``grow``
    (1 where the parent was live) and ``history`` (the parent, -1 where the beam has finished: :func:`kv_pages_update`'s parent), all int32.
    """
    shape, strides = logits.shape, logits.stride()
    if len(shape) != 2 or strides[1] != 1 and shape[1] > 1:
        raise InterpreterError(f"logits: {tuple(shape)}, expected [rows, vocabulary] with contiguous rows")
    rows, vocab = shape
    kind, n = _kind[logits.dtype], (rows,)
    if kind > _BF16:
        raise InterpreterError(f"logits: element type {_name(logits.dtype)}: float32, float16 or bfloat16")
    work, work_bytes = _scratch(scratch)
    _call("nc_beam_select",
          (_expect("parent", parent, _I32, n), _expect("tokens", tokens, _I64, n), _expect("new_scores", new_scores, _F32, n),
           0 if new_finished is None else _expect("new_finished", new_finished, _I32, n),
           0 if grow is None else _expect("grow", grow, _I32, n),
           0 if history is None else _expect("history", history, _I32, n),
           logits.data_ptr(), _expect("scores", scores, _F32, n),
           0 if finished is None else _expect("finished", finished, _I32, n),
           0 if norms is None else _expect("norms", norms, _F32, n), work, _error(error)),
          (rows, vocab, strides[0] if rows > 1 else vocab, kind, beams, end, work_bytes), stream)


_ITEM_BYTES = {_F32: 4, _F16: 2, _BF16: 2, _I32: 4, _I64: 8, _U64: 8, _U8: 1}


def _states(what: str, array) -> tuple[tuple, int, int]:
    """Shape ``(rows, planes, capacity, line)``, row stride and bytes of an element of states; rows may be strided."""
    shape, strides = tuple(array.shape), tuple(array.stride())
    if len(shape) == 2:
        shape, strides = (shape[0], 1, shape[1], 1), (strides[0], shape[1], strides[1], 1)
    size = _ITEM_BYTES.get(_kind[array.dtype])
    if len(shape) != 4 or size is None:
        raise InterpreterError(f"{what}: {_name(array.dtype)} {shape}, expected [rows, planes, positions, values] or [rows, positions]")
    rows, planes, capacity, line = shape
    for n, stride, expected in ((line, strides[3], 1), (capacity, strides[2], line), (planes, strides[1], capacity * line)):
        if n > 1 and stride != expected:
            raise InterpreterError(f"{what}: strides {strides}, expected contiguous rows")
    return shape, strides[0] if rows > 1 else planes * capacity * line, size


def beam_reorder(new, old, parent, *, lengths=None, new_lengths=None, append=None, grow=None, stream: int = 0) -> None:
    """States ``new[i] = old[parent[i]]``, up to the parent's length, and one position more from ``append`` (``nc_beam_reorder``).

    ``new`` and ``old``: ``[rows, planes, positions, values]`` or ``[rows, positions]`` of one type, not overlapping. ``lengths``
    (int32 ``[rows]``): the old rows' positions (default: all). ``append``: ``[rows, planes, values]`` or ``[rows]``, put at the end where
    ``grow`` (int32, default 1) is not 0. Rows with a parent outside ``0 .. rows - 1`` are left as they are.
    """
    shape, to_stride, size = _states("new", new)
    from_shape, from_stride, _ = _states("old", old)
    if from_shape != shape or _kind[old.dtype] != _kind[new.dtype]:
        raise InterpreterError(f"old: {_name(old.dtype)} {tuple(old.shape)}, expected new's {_name(new.dtype)} {tuple(new.shape)}")
    rows, planes, capacity, line = shape
    n = (rows,)
    tail = n if len(new.shape) == 2 else (rows, planes, line)
    _call("nc_beam_reorder",
          (new.data_ptr(), old.data_ptr(), _expect("parent", parent, _I32, n),
           0 if lengths is None else _expect("lengths", lengths, _I32, n),
           0 if new_lengths is None else _expect("new_lengths", new_lengths, _I32, n),
           0 if append is None else _expect("append", append, _kind[new.dtype], tail),
           0 if grow is None else _expect("grow", grow, _I32, n)),
          (rows, planes, capacity, line * size, to_stride * size, from_stride * size), stream)
