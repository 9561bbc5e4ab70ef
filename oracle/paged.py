"""Head norms with rotation, appends to and attention on a paged cache, restated in
numpy (test infrastructure). Everything is float64 from the inputs' values."""

from __future__ import annotations

import numpy as np

from .attention import attention_prefill


def rotate(x, cos_sin, positions, weight=None, eps=1e-6, offset=0, interleaved=False):
    """x [T, H, d], cos_sin [P, rotary], positions [T]. Returns the rotated heads and
    the size of what each value sums: |a c| + |b s|."""
    y = np.asarray(x, dtype=np.float64).copy()
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * np.asarray(weight, dtype=np.float64)
    size = np.abs(y)
    n = 0 if cos_sin is None else cos_sin.shape[1]
    if n:
        at = np.clip(positions, 0, cos_sin.shape[0] - 1)
        c, s = (np.asarray(t, dtype=np.float64)[at][:, None]
                for t in (cos_sin[:, :n // 2], cos_sin[:, n // 2:]))
        i = np.arange(n // 2)
        a, b = (offset + 2 * i, offset + 2 * i + 1) if interleaved else (offset + i, offset + n // 2 + i)
        ya, yb = y[..., a].copy(), y[..., b].copy()
        y[..., a], y[..., b] = ya * c - yb * s, yb * c + ya * s
        size[..., a], size[..., b] = np.abs(ya * c) + np.abs(yb * s), np.abs(yb * c) + np.abs(ya * s)
    return y, size


def bounds(cu, rows, sequences):
    """First row and number of new rows of each sequence."""
    if cu is None:
        n = rows // sequences
        return [(i * n, n) for i in range(sequences)]
    return [(int(a), int(b - a)) for a, b in zip(cu[:-1], cu[1:])]


def places(table, lengths, page_rows, pages, rows, cu=None):
    """Sequence (-1: none), position, page (-1: none) and row in it of each new row."""
    out = np.full((rows, 4), -1, dtype=np.int64)
    for s, (at, n) in enumerate(bounds(cu, rows, len(lengths))):
        length = max(int(lengths[s]), 0)
        for i in range(n):
            p = length - n + i
            out[at + i] = s, p, -1, -1
            if 0 <= p < table.shape[1] * page_rows and 0 <= table[s, p // page_rows] < pages:
                out[at + i, 2:] = table[s, p // page_rows], p % page_rows
    return out


def attention_paged(q, k_pages, v_pages, table, lengths, scale, cu=None):
    """q [T, H, dqk], pages [P, R, Hkv, d]: each sequence's positions gathered in order
    (zeros where there is no page, none beyond the table), then for each token the attention of
    dense keys, of which it sees those up to its own position. Returns its (out, spread, score)
    and the longest sequence."""
    page_rows = k_pages.shape[1]
    at = places(table, lengths, page_rows, k_pages.shape[0], q.shape[0], cu)[:, :2]
    most = table.shape[1] * page_rows
    keys, values = [], []
    for s, length in enumerate(lengths):
        length = min(max(int(length), 0), most)
        for pages, out in ((k_pages, keys), (v_pages, values)):
            rows = np.zeros((length, *pages.shape[2:]))
            for p in range(length):
                page = table[s, p // page_rows]
                if 0 <= page < pages.shape[0]:
                    rows[p] = pages[page, p % page_rows]
            out.append(rows)
    got = [np.zeros((*q.shape[:2], v_pages.shape[3])), np.zeros((*q.shape[:2], v_pages.shape[3])),
           np.zeros(q.shape[:2])]
    for i, (s, p) in enumerate(at):
        seen = min(p + 1, most)
        if s >= 0 and seen > 0:
            one = attention_prefill(q[i:i + 1], keys[s][:seen], values[s][:seen], scale)
            for t, x in zip(got, one):
                t[i] = x[0]
    return (*got, max((len(k) for k in keys), default=0))
