"""Forms of the paged-cache operators that small calls of a few heads do not reach: head norms and
appends of many rows (two a lane group, outputs past the caches), appends in fp16, heads of one key head
in several packs. Tolerances as in test_gpu_paged.py.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as P
from oracle.kda import round_to

from .test_gpu_paged import (DEV, _NAMES, _angles, _attend, _cache, _close, _cu, _head_bound, _np, _require_gpu, _t)

pytestmark = pytest.mark.gpu

_ = _require_gpu  # fixture


def _normal(rng, shape, dtype):
    return round_to(rng.normal(size=shape), _NAMES[dtype])


# tokens x heads pass 65536, 32768, 16384 and 8192 rows, from which on a call of that width is large
@pytest.mark.parametrize("tokens,h,hk,d,rotary,offset", [
    (9371, 5, 2, 64, 64, 0), (4691, 5, 2, 128, 64, 48), (2347, 4, 3, 256, 256, 0), (4999, 3, 4, 56, 24, 8),
    (2351, 5, 2, 104, 40, 24), (1187, 5, 2, 200, 72, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norms_and_rotation_of_many_rows(rng, tokens, h, hk, d, rotary, offset, interleaved, dtype):
    from local_kimi_amd.kernels import qk_norm_rope

    q, k = (_normal(rng, (tokens, n, d), dtype) for n in (h, hk))
    w = [_normal(rng, d, dtype) for _ in range(2)]
    cs, at = _angles(rng, 500, rotary), rng.integers(-3, 510, tokens)
    qt, kt, ct, pt = _t(q[None], dtype), _t(k[None], dtype), _t(cs, torch.float32), _t(at[None], torch.int32)
    wt, kw = [_t(x, dtype) for x in w], {"rotary_offset": offset, "interleaved": interleaved}
    got = qk_norm_rope(qt, kt, ct, pt, *wt, 1e-5, **kw)
    for x, y, weight in zip((q, k), got, w):
        want, size = P.rotate(x, cs, at, weight, 1e-5, offset, interleaved)
        _close(y, want, _head_bound(want, size, d, dtype))
    # the same in pieces, which are small calls, bit for bit
    step = 1000
    for i in range(0, tokens, step):
        piece = qk_norm_rope(qt[:, i:i + step], kt[:, i:i + step], ct, pt[:, i:i + step], *wt, 1e-5, **kw)
        assert torch.equal(piece[0], got[0][:, i:i + step]) and torch.equal(piece[1], got[1][:, i:i + step]), i


@pytest.mark.parametrize("tokens,h,hk,d,dv,rotary,offset,page_rows", [
    (9371, 3, 2, 64, 64, 64, 0, 64), (4691, 4, 2, 128, 128, 128, 0, 16), (1871, 5, 2, 192, 128, 64, 128, 64),
    (2351, 3, 2, 104, 40, 40, 24, 48), (1301, 3, 2, 64, 200, 16, 8, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_appends_of_many_rows(rng, tokens, h, hk, d, dv, rotary, offset, page_rows, dtype):
    """Sequences from none to thousands of new tokens; what is not theirs stays as it was."""
    from local_kimi_amd.kernels import paged_append, qk_norm_rope_append

    cuts = np.sort(rng.integers(0, tokens, 12))
    new = [int(n) for n in np.diff(np.concatenate(([0], cuts, [tokens])))]
    cached = [int(n) for n in rng.integers(0, 90, len(new))]
    cached[3] = -2  # two of its first tokens have no place
    lengths = [max(0, a + b) for a, b in zip(new, cached)]
    host, dev, table = _cache(rng, lengths, page_rows, hk, d, dv, dtype)
    rows = tokens + 3
    q, k, v = (_normal(rng, (rows, n, m), dtype) for n, m in ((h, d), (hk, d), (hk, dv)))
    w, cs, cu = [_normal(rng, d, dtype) for _ in range(2)], _angles(rng, 3000, rotary), _cu(new)
    at = P.places(table, lengths, page_rows, host[0].shape[0], rows, cu)
    has = at[:, 2] >= 0
    page, row = at[has, 2], at[has, 3]
    tl = (_t(table, torch.int32), _t(np.array(lengths), torch.int32))
    calls = {"cu_seqlens": _t(cu, torch.int32)}
    kt, vt = _t(k[None], dtype), _t(v[None], dtype)
    got = qk_norm_rope_append(_t(q[None], dtype), kt, vt, *dev, *tl, _t(cs, torch.float32),
                              *(_t(x, dtype) for x in w), 1e-6, rotary_offset=offset, **calls)
    want, size = P.rotate(q, cs, at[:, 1], w[0], 1e-6, offset)
    bound = _head_bound(want, size, d, dtype)
    want[at[:, 0] < 0] = 0.0
    _close(got, want, bound, "q")
    assert not got[0, tokens:].any()
    want, size = P.rotate(k, cs, at[:, 1], w[1], 1e-6, offset)
    full, limit = host[0].copy(), np.zeros_like(host[0])
    full[page, row], limit[page, row] = want[has], _head_bound(want, size, d, dtype)[has]
    _close(dev[0], full, limit + 1e-300, "k")
    values = host[1].copy()
    values[page, row] = v[has]
    assert np.array_equal(_np(dev[1]), values)
    paged_append(kt, vt, *dev, *tl, **calls)
    full = host[0].copy()
    full[page, row] = k[has]
    assert np.array_equal(_np(dev[0]), full) and np.array_equal(_np(dev[1]), values)


@pytest.mark.parametrize("h,hk,d,dv,rotary,offset,page_rows", [(4, 2, 128, 128, 128, 0, 16), (2, 2, 192, 128, 64, 128, 64),
                                                               (3, 1, 64, 40, 16, 8, 48), (1, 1, 16, 256, 16, 0, 16)])
@pytest.mark.parametrize("new,cached", [([1], [0]), ([1, 1, 1], [15, 0, 100]), ([40, 0, 1, 17], [3, 9, 64, 0])])
@pytest.mark.parametrize("interleaved", [False, True])
def test_appends_in_fp16(rng, h, hk, d, dv, rotary, offset, page_rows, new, cached, interleaved):
    from local_kimi_amd.kernels import paged_append, qk_norm_rope_append

    dtype = torch.float16
    lengths = [a + b for a, b in zip(new, cached)]
    host, dev, table = _cache(rng, lengths, page_rows, hk, d, dv, dtype, heads_first=interleaved)
    rows = sum(new) + 2
    q, k, v = (_normal(rng, (rows, n, m), dtype) for n, m in ((h, d), (hk, d), (hk, dv)))
    w, cs, cu = [_normal(rng, d, dtype) for _ in range(2)], _angles(rng, 128, rotary), _cu(new)
    at = P.places(table, lengths, page_rows, host[0].shape[0], rows, cu)
    page, row, n = at[:-2, 2], at[:-2, 3], sum(new)
    tl = (_t(table, torch.int32), _t(np.array(lengths), torch.int32))
    calls = {"cu_seqlens": _t(cu, torch.int32)}
    kt, vt = _t(k[None], dtype), _t(v[None], dtype)
    got = qk_norm_rope_append(_t(q[None], dtype), kt, vt, *dev, *tl, _t(cs, torch.float32),
                              *(_t(x, dtype) for x in w), 1e-6, rotary_offset=offset,
                              interleaved=interleaved, **calls)
    want, size = P.rotate(q, cs, at[:, 1], w[0], 1e-6, offset, interleaved)
    bound = _head_bound(want, size, d, dtype)
    want[n:] = 0.0
    _close(got, want, bound, "q")
    want, size = P.rotate(k, cs, at[:, 1], w[1], 1e-6, offset, interleaved)
    full, limit = host[0].copy(), np.zeros_like(host[0])
    full[page, row], limit[page, row] = want[:n], _head_bound(want, size, d, dtype)[:n]
    _close(dev[0], full, limit + 1e-300, "k")
    values = host[1].copy()
    values[page, row] = v[:n]
    assert np.array_equal(_np(dev[1]), values)
    paged_append(kt, vt, *dev, *tl, **calls)
    full = host[0].copy()
    full[page, row] = k[:n]
    assert np.array_equal(_np(dev[0]), full) and np.array_equal(_np(dev[1]), values)


# packs of 32, 17 (two units of 16 rows, the second in part), 1, 27 and 32, one or more a key head
@pytest.mark.parametrize("h,hk", [(64, 1), (34, 1), (37, 1), (54, 2), (128, 2)])
@pytest.mark.parametrize("dq,dv", [(64, 64), (192, 128)])
@pytest.mark.parametrize("new,cached", [([1], [0]), ([1, 1, 1, 1], [0, 63, 64, 130]), ([5, 0, 2], [100, 9, 0]),
                                        ([37, 1, 60], [0, 300, 45])])
def test_several_packs_of_heads_on_a_key_head(rng, h, hk, dq, dv, new, cached):
    _attend(rng, new, cached, 16, h, hk, dq, dv, torch.bfloat16)


@pytest.mark.parametrize("h,hk", [(64, 1), (34, 1), (37, 1), (54, 2)])
@pytest.mark.parametrize("new,cached", [([1, 1], [1500, 2]), ([1, 30, 1], [900, 800, 2])])
def test_several_packs_on_long_caches_in_runs(rng, h, hk, new, cached):
    _attend(rng, new, cached, 16, h, hk, 128, 128, torch.float16)


def test_many_sequences_of_several_packs(rng):
    """Beyond 256 sequences, where a launch of its own counts through them."""
    new = [int(n) for n in rng.integers(0, 3, 260)]
    cached = [int(n) for n in rng.integers(0, 20, 260)]
    cached[100], new[100] = 900, 1
    _attend(rng, new, cached, 16, 34, 1, 64, 64, torch.bfloat16)
