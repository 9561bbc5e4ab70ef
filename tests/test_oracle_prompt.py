"""The oracles of the prompt operators (oracle/kda.py, oracle/attention.py) against
hand-computed cases, other formulations and planted mistakes; CPU only."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kda as K
from oracle.attention import attention_prefill


def test_sequence_bounds_clamp_and_divide():
    assert K.sequence_bounds(None, 6, 3) == [(0, 2), (2, 4), (4, 6)]
    assert K.sequence_bounds(np.array([0, 2, 2, 9]), 6, 3) == [(0, 2), (2, 2), (2, 6)]
    assert K.sequence_bounds(np.array([0, 5, 3, -4]), 6, 3) == [(0, 5), (5, 5), (3, 3)]


def test_short_conv_prefill_is_a_causal_convolution(rng):
    """Against torch's conv1d over (state[1:], tokens), per sequence."""
    c, cu = 5, np.array([0, 3, 3, 4, 11])
    x, w = rng.normal(size=(13, c)), rng.normal(size=(c, 1, 4))
    st = rng.normal(size=(4, c, 4))
    out, new = K.short_conv_prefill(x, st, w, "float32", cu)
    for s in range(4):
        a, b = cu[s], cu[s + 1]
        line = np.concatenate((st[s].T, x[a:b]))
        assert np.array_equal(new[s], line[-4:].T)
        if b > a:
            y = torch.nn.functional.conv1d(torch.from_numpy(line[1:].T.copy())[None],
                                           torch.from_numpy(w), groups=c)[0].T
            want = torch.nn.functional.silu(y).numpy()
            assert np.allclose(out[a:b], want, rtol=1e-6, atol=1e-6)
    assert not out[11:].any()


def _solve_scan(state, q, k, v, decay, beta, scale):
    """The recurrence of one head as one triangular solve (another formulation)."""
    g = np.cumsum(decay, 0)
    t = q.shape[0]
    a, p = np.eye(t), np.zeros((t, t))
    for i in range(t):
        for j in range(i + 1):
            e = k[j] * np.exp(g[i] - g[j]) * beta[j]
            p[i, j] = q[i] @ e
            if j < i:
                a[i, j] = k[i] @ e
    u = np.linalg.solve(a, v - (k * np.exp(g)) @ state)
    out = scale * ((q * np.exp(g)) @ state + p @ u)
    new = np.exp(g[-1])[:, None] * state + (k * np.exp(g[-1] - g) * beta[:, None]).T @ u
    return new, out


def _scan_inputs(rng, t, h, dk, dv, n):
    q, k = rng.normal(size=(2, t, h, dk))
    q /= np.linalg.norm(q, axis=-1, keepdims=True)
    k /= np.linalg.norm(k, axis=-1, keepdims=True)
    return (rng.normal(size=(n, h, dk, dv)), q, k, rng.normal(size=(t, h, dv)),
            -rng.uniform(0, 0.5, size=(t, h, dk)), rng.uniform(size=(t, h)))


def test_prefill_equals_the_triangular_solve(rng):
    cu = np.array([0, 7, 7, 20])
    state, q, k, v, decay, beta = _scan_inputs(rng, 21, 2, 6, 5, 3)
    new, out = K.prefill(state, q, k, v, decay, beta, 0.3, cu)
    for s in (0, 2):
        a, b = cu[s], cu[s + 1]
        for h in range(2):
            want_s, want_o = _solve_scan(state[s, h], q[a:b, h], k[a:b, h], v[a:b, h],
                                         decay[a:b, h], beta[a:b, h], 0.3)
            assert np.allclose(new[s, h], want_s, atol=1e-12)
            assert np.allclose(out[a:b, h], want_o, atol=1e-12)
    assert np.array_equal(new[1], state[1]) and not out[20:].any()


def test_a_planted_mistake_fails_the_triangular_solve(rng):
    """Decay after the correction instead of before it is another function."""
    state, q, k, v, decay, beta = _scan_inputs(rng, 9, 1, 6, 5, 1)
    want, _ = _solve_scan(state[0, 0], q[:, 0], k[:, 0], v[:, 0], decay[:, 0], beta[:, 0], 1.0)
    s = state[0, 0].copy()
    for t in range(9):
        s = s + beta[t, 0] * np.outer(k[t, 0], v[t, 0] - s.T @ k[t, 0])
        s = s * np.exp(decay[t, 0])[:, None]
    assert not np.allclose(s, want, atol=1e-3)


def test_attention_hand_computed():
    """Two queries, unit scores: the first sees v0, the second the mean."""
    q = np.ones((2, 1, 8))
    k = np.zeros((2, 1, 8))
    v = np.stack([np.full((1, 8), 2.0), np.full((1, 8), 4.0)])
    out, spread, score = attention_prefill(q, k, v, 1.0)
    assert np.array_equal(out[:, 0, 0], [2.0, 3.0]) and np.array_equal(spread, out)
    assert not score.any()


@pytest.mark.parametrize("lq,lk", [(5, 5), (3, 9), (6, 2)])
def test_attention_matches_torch(rng, lq, lk):
    q, k, v = rng.normal(size=(lq, 4, 8)), rng.normal(size=(lk, 2, 8)), rng.normal(size=(lk, 2, 16))
    out, _, _ = attention_prefill(q, k, v, 0.4)
    tq, tk, tv = (torch.from_numpy(x).transpose(0, 1) for x in (q, k, v))
    mask = torch.ones(lq, lk, dtype=torch.bool).tril(lk - lq)
    s = (0.4 * tq @ tk.repeat_interleave(2, 0).transpose(1, 2)).masked_fill(~mask, -np.inf)
    want = torch.nan_to_num(torch.softmax(s, -1)) @ tv.repeat_interleave(2, 0)
    assert np.allclose(out, want.transpose(0, 1).numpy(), atol=1e-12)


def test_attention_leaves_unseen_rows_out(rng):
    """NaN and infinity behind a query, and in another sequence, change nothing."""
    q, k, v = (rng.normal(size=(6, 2, 8)) for _ in range(3))
    cu = np.array([0, 4, 6])
    out, _, _ = attention_prefill(q, k, v, 1.0, 2, cu, cu)
    k2, v2 = k.copy(), v.copy()
    k2[3], v2[3] = np.nan, np.inf
    out2, _, _ = attention_prefill(q, k2, v2, 1.0, 2, cu, cu)
    assert np.array_equal(out[:3], out2[:3]) and np.array_equal(out[4:], out2[4:])
    assert np.isnan(out2[3]).all()
