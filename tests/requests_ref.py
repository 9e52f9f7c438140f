"""Plain NumPy forms, in 64 bits, of low-rank adapters, beam selection and reordering of states, for the tests."""

from __future__ import annotations

import numpy as np


def lora(x, a, b, widths, rank, adapters, row_start, base=None, ranks=None, scales=None):
    """Outputs [rows, outputs], and a bound on what float32 sums lose: rows and sums in two parts of 11 bits lose 2^-24 of
    a term, a chain of eight matrix instructions 2^-22 of its terms' sum each (they cut off), further additions 2^-24 each."""
    rows = x.shape[0]
    out = np.zeros((rows, sum(widths))) if base is None else base.astype(np.float64)
    bound = np.zeros_like(out)
    x, a, b = (v.astype(np.float64) for v in (x, a, b))
    inputs = x.shape[1]
    of_h, of_out = (2.0 ** -24 * (34 + n / 32 + 16) for n in (inputs, rank))
    for i, s in enumerate(adapters):
        at = slice(row_start[i], row_start[i + 1])
        if not 0 <= s < a.shape[0] or row_start[i + 1] <= row_start[i]:
            continue
        r = rank if ranks is None else int(np.clip(ranks[s], 0, rank))
        scale = 1.0 if scales is None else float(scales[s])
        n = 0
        for t, w in enumerate(widths):
            first, second = a[s, t * rank: t * rank + r], b[s, n: n + w, :r]
            with np.errstate(all="ignore"):
                h, h_size = x[at] @ first.T, np.abs(x[at]) @ np.abs(first).T
                out[at, n: n + w] += scale * (h @ second.T)
                bound[at, n: n + w] = abs(scale) * ((of_h * h_size + of_out * np.abs(h)) @ np.abs(second).T)
            n += w
    return out, bound


def beams(logits, scores, width, end=-1, finished=None, norms=None):
    """Each request's candidates in their order: parent, token, total, rank value; then the outputs of a choice."""
    rows, vocab = logits.shape
    finished = np.zeros(rows, np.int32) if finished is None else finished
    norms = np.ones(rows) if norms is None else norms.astype(np.float64)
    x = logits.astype(np.float64)
    chosen = []
    for first in range(0, rows, width):
        found = []
        for r in range(first, first + width):
            s = float(scores[r])
            if np.isnan(s) or s == -np.inf:
                continue
            if finished[r]:
                found.append((s / norms[r], r, end, s, True))
                continue
            most = x[r].max()
            if not most < np.inf or most == -np.inf:
                continue
            lse = most + np.log(np.exp(x[r] - most).sum())
            for v in np.argsort(-x[r], kind="stable")[:width]:
                if x[r, v] > -np.inf:
                    total = s + (x[r, v] - lse)
                    found.append((total / norms[r], r, int(v), total, False))
        found.sort(key=lambda c: -c[0])                              # stable: the lower row first, then the row's own order
        chosen.append(found)
    return chosen


def beam_outputs(found, width, end):
    """parent, token, total, finished, grow, history of the best `width` of a request's candidates."""
    out = []
    for i in range(width):
        if i >= len(found):
            out.append((-1, max(end, 0), -np.inf, 1, 0, -1))
            continue
        _, row, token, total, was = found[i]
        over = was or (end >= 0 and token == end)
        out.append((row, token, total, int(over), int(not was), -1 if over else row))
    return out


def reorder(new, old, parent, lengths=None, append=None, grow=None):
    """new [rows, planes, positions, values] after the call, and the new lengths."""
    new = new.copy()
    rows, _, capacity, _ = new.shape
    after = np.zeros(rows, np.int32)
    for i, p in enumerate(parent):
        if not 0 <= p < rows:
            continue
        n = capacity if lengths is None else int(np.clip(lengths[p], 0, capacity))
        new[i, :, :n] = old[p, :, :n]
        if append is not None and n < capacity and (grow is None or grow[i]):
            new[i, :, n] = append[i]
            n += 1
        after[i] = n
    return new, after
