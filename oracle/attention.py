"""Causal attention of packed prompts, restated in numpy (test infrastructure).

Only the tests use this module, as the checker of the HIP kernel; nothing in
the product path calls it. Everything is float64 from the inputs' values.
"""

from __future__ import annotations

import numpy as np

from .kda import sequence_bounds


def attention_prefill(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float,
                      sequences: int = 1, cu_q: np.ndarray | None = None,
                      cu_k: np.ndarray | None = None) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """q [T, H, dqk], k [Tk, Hkv, dqk], v [Tk, Hkv, dv]: query i of a sequence of
    lq queries and lk keys sees keys 0 .. i + lk - lq; what it does not see is
    left out of its sums altogether. Returns (out, spread, score): the output
    [T, H, dv] (zeros for a query that sees nothing and for rows of no
    sequence), sum p |v| of each output, and the largest scale * sum |q| |k|
    over each query's keys [T, H]: what the rounding of p and of the scores
    can move."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    heads, group = q.shape[1], q.shape[1] // k.shape[1]
    out = np.zeros((q.shape[0], heads, v.shape[2]))
    spread, score = np.zeros_like(out), np.zeros(q.shape[:2])
    for (qa, qb), (ka, kb) in zip(sequence_bounds(cu_q, q.shape[0], sequences),
                                  sequence_bounds(cu_k, k.shape[0], sequences)):
        for i in range(qb - qa):
            seen = min(kb - ka, i + (kb - ka) - (qb - qa) + 1)
            if seen <= 0:
                continue
            for h in range(heads):
                kk, vv = k[ka:ka + seen, h // group], v[ka:ka + seen, h // group]
                s = scale * (kk @ q[qa + i, h])
                p = np.exp(s - s.max())
                p /= p.sum()
                out[qa + i, h] = p @ vv
                spread[qa + i, h] = p @ np.abs(vv)
                score[qa + i, h] = abs(scale) * (np.abs(kk) @ np.abs(q[qa + i, h])).max()
    return out, spread, score
