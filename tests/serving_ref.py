"""Plain NumPy forms of the serving operators, in 64 bits where they sum, for the tests.

The cache's layout and rounding steps are restated here from their definition (``nc_kv4.cuh``): codes and
parameters are found by position, head and dimension, one at a time.
"""

from __future__ import annotations

import numpy as np

BF16 = "bfloat16"


def to_bf16(x: np.ndarray) -> np.ndarray:
    """float32 to the uint16 bits of bfloat16, to nearest even (NaN kept)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u >> 16) + (((u & 0xFFFF) > 0x8000) | (((u & 0xFFFF) == 0x8000) & ((u >> 16) & 1)))).astype(np.uint32)
    return np.where(np.isnan(x), 0x7FC0, r).astype(np.uint16)


def from_bf16(u: np.ndarray) -> np.ndarray:
    return (u.astype(np.uint32) << 16).view(np.float32)


def encode(x: np.ndarray, dtype: str) -> np.ndarray:
    """float32 values as the host array of a device array of ``dtype``."""
    return to_bf16(x) if dtype == BF16 else x.astype(dtype)


def decode(x: np.ndarray, dtype: str) -> np.ndarray:
    return from_bf16(x) if dtype == BF16 else x.astype(np.float32)


def rope_tables(positions: int, d: int) -> tuple[np.ndarray, np.ndarray]:
    angles = np.arange(positions)[:, None] * (1e4 ** (-np.arange(0, d, 2) / d))[None]
    return np.cos(angles).astype(np.float32), np.sin(angles).astype(np.float32)


def rotate(x: np.ndarray, position: np.ndarray, rope) -> np.ndarray:
    """Rows ``x`` [rows, heads, d] rotated by their positions, in ``x``'s precision, each operation rounded."""
    if rope is None:
        return x
    cos, sin = (t[np.maximum(position, 0)][:, None].astype(x.dtype) for t in rope)
    a, b = np.split(x, 2, axis=-1)
    return np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """float32 [..., d] to codes [..., d / 32, 32], scale and zero [..., d / 32] (float16)."""
    x = x.reshape(*x.shape[:-1], -1, 32).astype(np.float32)
    with np.errstate(all="ignore"):
        low, high = x.min(-1), x.max(-1)
        nan = np.isnan(low) | np.isnan(high)
        limit = np.float32(65504)
        zero = np.clip(low, -limit, limit)
        width = (high - low) * np.float32(1 / 15)
        scale = np.where(np.isnan(width) & ~nan, limit, np.minimum(width, limit))
        zero, scale = (np.where(nan, np.nan, v).astype(np.float16) for v in (zero, scale))
        s = scale.astype(np.float32)[..., None]
        code = np.floor((x - zero.astype(np.float32)[..., None]) * (np.float32(1) / np.where(s > 0, s, np.float32(1))) + np.float32(0.5))
        code = np.where(s > 0, np.clip(code, 0, 15), 0)
    return code.astype(np.uint8), scale, zero


def stands_for(code, scale, zero) -> np.ndarray:
    """The float32 values that codes stand for, [..., d]."""
    with np.errstate(all="ignore"):
        v = zero.astype(np.float32)[..., None] + scale.astype(np.float32)[..., None] * code.astype(np.float32)
    return v.reshape(*v.shape[:-2], -1)


class Pool:
    """A pool's bytes: [pages, layers * kv * page * d * 5 / 4] uint8, read and written by position."""

    def __init__(self, pages: int, kv: int, d: int, page: int, layers: int = 1, fill: int = 0xFF):
        self.kv, self.d, self.page, self.layers = kv, d, page, layers
        self.layer_bytes = kv * page * d * 5 // 4
        self.bytes = np.full((pages, layers * self.layer_bytes), fill, np.uint8)

    def _tile(self, page_id: int, layer: int, head: int, inside: int) -> np.ndarray:
        start = layer * self.layer_bytes + (head * (self.page // 16) + inside // 16) * 20 * self.d
        return self.bytes[page_id, start: start + 20 * self.d]

    def put(self, page_id: int, layer: int, head: int, inside: int, which: int, code, scale, zero) -> None:
        """One position's row: codes [d / 32, 32], scale and zero [d / 32]; ``which``: 0 keys, 1 values."""
        nb = self.d // 32
        vb = 2 if nb % 2 == 0 else 1
        t = inside % 16
        j, g, c, h = t // 8, t % 8, t % 8 // 2, t % 2
        half = self._tile(page_id, layer, head, inside)[which * 10 * self.d:]
        words, shorts = half[: 8 * self.d].view(np.uint32), half[: 8 * self.d].view(np.uint16)
        params = half[8 * self.d: 10 * self.d].view(np.float16).reshape(8, nb, 2, 2)
        for b in range(nb):
            params[g, b, j] = scale[b], zero[b]
            if which == 0:
                for cc in range(4):
                    word = sum(int(code[b, 8 * cc + i]) << 4 * i for i in range(8))
                    words[(((b // vb * 8 + g) * 4 + cc) * vb + b % vb) * 2 + j] = word
            else:
                for gg in range(8):
                    short = sum(int(code[b, 4 * gg + i]) << 4 * i for i in range(4))
                    shorts[((((b // vb * 8 + gg) * 4 + c) * vb + b % vb) * 2 + j) * 2 + h] = short

    def get(self, page_id: int, layer: int, head: int, inside: int, which: int) -> np.ndarray:
        """The float32 values [d] of one position."""
        nb = self.d // 32
        vb = 2 if nb % 2 == 0 else 1
        t = inside % 16
        j, g, c, h = t // 8, t % 8, t % 8 // 2, t % 2
        half = self._tile(page_id, layer, head, inside)[which * 10 * self.d:]
        words, shorts = half[: 8 * self.d].view(np.uint32), half[: 8 * self.d].view(np.uint16)
        params = half[8 * self.d: 10 * self.d].view(np.float16).reshape(8, nb, 2, 2)
        code = np.empty((nb, 32), np.uint8)
        for b in range(nb):
            for i in range(32):
                if which == 0:
                    code[b, i] = words[(((b // vb * 8 + g) * 4 + i // 8) * vb + b % vb) * 2 + j] >> 4 * (i % 8) & 15
                else:
                    code[b, i] = shorts[((((b // vb * 8 + i // 4) * 4 + c) * vb + b % vb) * 2 + j) * 2 + h] >> 4 * (i % 4) & 15
        return stands_for(code, params[g, :, j, 0], params[g, :, j, 1])

    def append(self, keys, values, table, lengths, row_start, rope=None, layer: int = 0) -> None:
        """Rows ``keys`` and ``values`` (float32 [rows, kv, d]) as the sequences' last positions."""
        for i, length in enumerate(lengths):
            rows = range(row_start[i], row_start[i + 1])
            for r in rows:
                position = length - (row_start[i + 1] - r)
                if position < 0:
                    continue
                k = rotate(keys[r: r + 1], np.array([position]), rope)[0]
                for which, x in ((0, k), (1, values[r])):
                    code, scale, zero = quantise(x)
                    for head in range(self.kv):
                        self.put(table[i, position // self.page], layer, head, position % self.page, which, code[head],
                                 scale[head], zero[head])

    def history(self, table_row, length: int, layer: int = 0) -> tuple[np.ndarray, np.ndarray]:
        """The keys and values of a sequence, [length, kv, d] float32."""
        out = np.empty((2, length, self.kv, self.d), np.float32)
        for t in range(length):
            for which in range(2):
                for head in range(self.kv):
                    out[which, t, head] = self.get(table_row[t // self.page], layer, head, t % self.page, which)
        return out[0], out[1]


def attention(q, histories, lengths, row_start, scale, rope=None):
    """Rows ``q`` [rows, heads, d] over (keys, values) [length, kv, d] of each sequence, in 64 bits: the output
    [rows, heads, d], the log-sums [rows, heads], and sum_i |q_i k_i| at its largest over what each row and head sees."""
    rows, heads, d = q.shape
    out = np.zeros((rows, heads, d))
    lse = np.full((rows, heads), -np.inf)
    size = np.zeros((rows, heads))
    for i, length in enumerate(lengths):
        keys, values = (x.astype(np.float64) for x in histories[i])
        for r in range(row_start[i], row_start[i + 1]):
            position = length - (row_start[i + 1] - r)
            if position < 0:
                continue
            x = rotate(q[r: r + 1].astype(np.float64), np.array([position]), rope)[0]
            for h in range(heads):
                head = h // (heads // keys.shape[1])
                k, v = keys[: position + 1, head], values[: position + 1, head]
                s = k @ x[h] * scale
                m = s.max()
                p = np.exp(s - m)
                out[r, h] = p @ v / p.sum()
                lse[r, h] = m + np.log(p.sum())
                size[r, h] = (np.abs(k) @ np.abs(x[h])).max() * scale
    return out, lse, size


def pages_update(table, lengths, page: int, pages: int, parent=None, grow=None):
    """New table, lengths, status and the copied pages [(from, to)], one sequence and page at a time."""
    seqs, width = table.shape
    parent = np.arange(seqs) if parent is None else parent
    grow = np.zeros(seqs, int) if grow is None else grow
    kept, after, refs = [], [], {}
    for i in range(seqs):
        p = parent[i] if 0 <= parent[i] < seqs else -1
        before = 0 if p < 0 else max(0, int(lengths[p]))
        n = 0 if p < 0 else min(max(before + int(grow[i]), 0), width * page)
        kept.append(min(before, n))
        after.append(n)
        for j in range(-(-kept[i] // page)):
            if not 0 <= table[p, j] < pages:
                return table.copy(), lengths.copy(), [-1, 0, 0, 0], []
            refs.setdefault(int(table[p, j]), []).append((i, j == kept[i] // page and kept[i] % page != 0))
    free = iter([x for x in range(pages) if x not in refs])
    new = np.full_like(table, -1)
    copies, missing, fresh = [], 0, 0
    for i in range(seqs):
        for j in range(-(-after[i] // page)):
            old = int(table[parent[i], j]) if j < -(-kept[i] // page) else None
            if old is not None:
                is_tail = j == kept[i] // page and kept[i] % page != 0
                users = refs[old]
                mine = not is_tail or (all(t for _, t in users) and min(u for u, _ in users) == i)
                if mine:
                    new[i, j] = old
                    continue
            page_id = next(free, None)
            if page_id is None:
                missing += 1
                continue
            fresh += 1
            new[i, j] = page_id
            if old is not None:
                copies.append((old, page_id))
    if missing:
        used = {int(table[i, j]) for i in range(seqs) for j in range(-(-max(0, int(lengths[i])) // page))
                if j < width and 0 <= table[i, j] < pages}
        return table.copy(), lengths.copy(), [missing, len(used), 0, 0], []
    highest = int(new.max()) + 1 if new.size else 0
    return new, np.array(after, np.int32), [0, len(refs) + fresh, len(copies), highest], copies


def pages_compact(table, lengths, page: int, pages: int):
    seqs, width = table.shape
    live = {int(table[i, j]) for i in range(seqs) for j in range(-(-max(0, int(lengths[i])) // page)) if j < width}
    if any(not 0 <= x < pages for x in live):
        return table.copy(), [-1, 0, 0, 0], []
    n = len(live)
    moves = list(zip(sorted(x for x in live if x >= n), sorted(set(range(n)) - live)))
    to = dict(moves)
    new = np.full_like(table, -1)
    for i in range(seqs):
        for j in range(-(-max(0, int(lengths[i])) // page)):
            if j < width:
                new[i, j] = to.get(int(table[i, j]), int(table[i, j]))
    return new, [0, n, len(moves), n], moves


def logprobs(x, targets, k: int):
    """Log probabilities of ``targets``, entropy, log-sums, top ids and their log probabilities, in 64 bits."""
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        m = x.max(-1, keepdims=True)
        none = np.isneginf(m[:, 0])
        c = x - np.where(np.isneginf(m), 0, m)
        e = np.exp(c)
        total = e.sum(-1)
        log_total = np.log(total)
        logp = c - log_total[:, None]
        logp[none] = -np.inf
        entropy = np.where(none, 0, log_total - np.where(e > 0, e * c, 0).sum(-1) / total)
        entropy = np.where(np.isnan(m[:, 0]), np.nan, entropy)
        lse = np.where(none, -np.inf, m[:, 0] + log_total)
    order = np.empty((x.shape[0], k), np.int64)
    for r in range(x.shape[0]):
        key = np.where(np.isnan(x[r]), np.inf, x[r])
        order[r] = np.lexsort((np.arange(x.shape[1]), -key, ~np.isnan(x[r])))[:k]
    rows = np.arange(x.shape[0])[:, None]
    return logp[rows, targets], entropy, lse, order, logp[rows, order]
