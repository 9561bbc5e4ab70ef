"""Lengths beyond what the table can name: a token keeps its position, and attends to the
positions up to it that the table names. Tolerances as in test_gpu_paged.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as P
from oracle.kda import round_to

from .test_gpu_paged import DEV, _NAMES, _cache, _close, _cu, _np, _require_gpu, _t

pytestmark = pytest.mark.gpu

_ = _require_gpu  # fixture


# new tokens, and positions beyond the table (which names 3 pages or more) by each length
@pytest.mark.parametrize("new,beyond", [([3], [2]), ([3, 1, 4], [3, 1, 0]), ([1, 5], [40, 5]),
                                        ([40, 1], [17, 0]), ([150, 33], [60, 200]), ([100, 2], [2 ** 30, 2 ** 31])])
@pytest.mark.parametrize("h,hk,dq,dv", [(4, 1, 128, 128), (2, 2, 192, 128), (32, 1, 64, 64)])
@pytest.mark.parametrize("cached", [40, 1000])
def test_tokens_keep_their_positions(rng, new, beyond, h, hk, dq, dv, cached):
    from local_kimi_amd.kernels import attention_paged, paged_append

    dtype, page_rows = torch.bfloat16, 16
    named = [cached + n for n in new]
    host, dev, table = _cache(rng, named, page_rows, hk, dq, dv, dtype)
    table = table[:, :-1]  # as wide as the longest
    most = table.shape[1] * page_rows
    lengths = np.array([min(most + b, 2 ** 31 - 1) for b in beyond])
    for s in range(len(new)):  # (pages without a sequence's own are shared: reads alone)
        table[s][table[s] < 0] = table[s, 0]
    cu = _cu(new)
    q = round_to(rng.normal(size=(sum(new), h, dq)), _NAMES[dtype])
    args = (_t(q[None], dtype), *dev, _t(table, torch.int32))
    kw = {"cu_seqlens": _t(cu, torch.int32)}
    got = attention_paged(*args, _t(lengths, torch.int32), **kw)
    want, spread, score, keys = P.attention_paged(q, *host, table, lengths, dq ** -0.5, cu)
    half = torch.finfo(dtype).eps / 2
    fp32 = 2.0 ** -24 * (2 * (dq + 8) * score[..., None] + keys + 8) * spread
    _close(got, want, half * (1 + half) * (spread + np.abs(want)) + 1.1 * fp32 + 2.0 ** -25,
           f"{new} beyond {beyond}")
    assert torch.equal(got, attention_paged(*args, _t(lengths, torch.int64), **kw))
    if cached > 100:
        return
    # new values of one on a cache of zeros, scores of zero: the share of the new ones among what a
    # token sees; p, its sums and those of the values are whole numbers, so that two roundings remain
    table = np.arange(table.size, dtype=np.int32).reshape(table.shape)
    own = [torch.zeros((table.size, *t.shape[1:]), dtype=dtype, device=DEV) for t in dev]
    tl = _t(table, torch.int32), _t(lengths, torch.int32)
    q0 = torch.zeros_like(args[0])
    paged_append(q0[:, :, :hk], torch.ones((1, sum(new), hk, dv), dtype=dtype, device=DEV), *own, *tl, **kw)
    got = _np(attention_paged(q0, *own, *tl, **kw))
    for s, (a, n) in enumerate(P.bounds(cu, sum(new), len(new))):
        first = int(lengths[s]) - n
        for i in range(n):
            seen = min(first + i + 1, most)
            share = max(0, seen - first) / seen
            assert np.all(np.abs(got[0, a + i] - share) <= (2.0 ** -8 + 2.0 ** -22) * share), (s, i)
