"""GPU parity of the paged-cache operators (local_kimi_amd/csrc/paged_cache.hip,
paged_attention.hip) with oracle/paged.py.

Tolerances, element by element against float64 on the same inputs. Heads: the mean
of d squares in fp32 is off by at most (d / 2 + 2) * 2^-24 relative (sums of squares, none
cancels, at worst one after the other over half the values and the lanes), its inverse root by half
of that and three roundings, x r w and the product with cos or sin by three more, their sum by one:
(d / 4 + 12) * 2^-24 of |a c| + |b s|, then one rounding to the type (eps / 2; fp16 below 2^-14
2^-25). Attention: as for dense keys (tests/test_gpu_attention.py), eps / 2 of sum p |v| for
the rounding of p, eps / 2 of the output, scores off by (d_qk + 8) * 2^-24 of scale * sum |q| |k|,
twice that in p, sums by 2^-24 a key.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as P
from oracle.kda import round_to

pytestmark = pytest.mark.gpu

DEV = "cuda"
_NAMES = {torch.float16: "float16", torch.bfloat16: "bfloat16", torch.float32: "float32"}


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from local_kimi_amd import _lib

    _lib.load()


def _t(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV, dtype)


def _np(t):
    return t.detach().double().cpu().numpy()


def _cu(lengths):
    return np.concatenate(([0], np.cumsum(lengths))).astype(np.int32)


def _angles(rng, rows, rotary):
    a = rng.uniform(0, 6.3, (rows, rotary // 2))
    return np.concatenate((np.cos(a), np.sin(a)), 1).astype(np.float32)


def _head_bound(y, size, d, dtype):
    half = torch.finfo(dtype).eps / 2
    return half * np.abs(y) + (1 + half) * 2.0 ** -24 * (d / 4 + 12) * size + \
        (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)


def _close(got, want, bound, what=""):
    g = _np(got).reshape(want.shape)
    err = np.abs(g - want)
    assert np.isfinite(g).all() and np.all(err <= bound), f"{what}: {np.max(err / bound):.3f} of the bound"


# ---------------------------------------------------------------------------
# norms and rotation


@pytest.mark.parametrize("h,hk,d,rotary,offset", [(4, 2, 128, 128, 0), (3, 1, 192, 64, 128),
                                                  (2, 2, 64, 32, 0), (5, 5, 8, 8, 0),
                                                  (1, 3, 256, 256, 0), (6, 2, 104, 40, 24)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norms_and_rotation_match_oracle(rng, h, hk, d, rotary, offset, interleaved, dtype):
    from local_kimi_amd.kernels import qk_norm_rope

    cs = _angles(rng, 50, rotary)
    for rows, norm, wide in ((1, True, False), (7, True, True), (37, False, False), (300, True, True)):
        q, k = (round_to(rng.normal(size=(rows, n, d)), _NAMES[dtype]) for n in (h, hk))
        w = [round_to(1 + 0.3 * rng.normal(size=d), _NAMES[dtype]) if norm else None for _ in range(2)]
        wt = [x if x is None else _t(x, torch.float32 if wide else dtype) for x in w]
        at = rng.integers(-3, 60, rows)
        got = qk_norm_rope(_t(q[None], dtype), _t(k[None], dtype), _t(cs, torch.float32),
                           _t(at[None], torch.int64 if wide else torch.int32), *wt, 1e-5,
                           rotary_offset=offset, interleaved=interleaved)
        for x, y, weight in zip((q, k), got, w):
            want, size = P.rotate(x, cs, at, weight, 1e-5, offset, interleaved)
            assert y.dtype == dtype and y.is_contiguous()
            _close(y, want, _head_bound(want, size, d, dtype), f"{rows} {norm}")


def test_heads_of_zeros_and_of_one_large_value():
    """A head of zeros stays zeros (eps alone under the root), one of a single value x
    becomes sqrt(d) w there; positions beyond the table are its last."""
    from local_kimi_amd.kernels import qk_norm_rope

    q = torch.zeros((1, 2, 1, 64), device=DEV)
    q[0, 1, 0, 9] = -3e15
    cs = torch.zeros((4, 64), device=DEV)
    cs[:, :32] = 1.0
    cs[3] = 0.0
    cs[3, 32:] = 1.0  # the last position: a quarter turn
    w = torch.full((64,), 2.0, device=DEV)
    got, _ = qk_norm_rope(q, q, cs, torch.tensor([[0, 0]], device=DEV), w, w)
    assert not got[0, 0].any() and abs(got[0, 1, 0, 9].item() + 16) < 16 * 2 ** -20
    got, _ = qk_norm_rope(q, q, cs, torch.tensor([[99, 2 ** 40]], device=DEV), w, w)
    assert abs(got[0, 1, 0, 41].item() + 16) < 16 * 2 ** -20 and not got[0, 1, 0, 9].any()


def test_strided_heads_and_batches(rng):
    from local_kimi_amd.kernels import qk_norm_rope

    fused = torch.randn((3, 11, 10, 72), device=DEV).bfloat16()
    q, k = fused[:, :, :6, :64], fused[:, :, 6:, :64]
    cs = _t(_angles(rng, 40, 64), torch.float32)
    at = torch.arange(33, device=DEV).reshape(3, 11)
    w = torch.rand(64, device=DEV).bfloat16()
    want = qk_norm_rope(q.contiguous(), k.contiguous(), cs, at, w, w)
    odd = torch.zeros((3, 11, 6, 65), device=DEV).bfloat16()[..., 1:]
    odd.copy_(q)
    for a in (q, odd, q.transpose(1, 2).contiguous().transpose(1, 2)):
        got = qk_norm_rope(a, k, cs, at.int(), w, w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = torch.zeros((1, 0, 6, 64), device=DEV)
    assert qk_norm_rope(one, one, cs, torch.zeros((1, 0), dtype=torch.int32, device=DEV))[0].shape == one.shape


# ---------------------------------------------------------------------------
# caches


def _cache(rng, lengths, page_rows, hk, d_qk, d_v, dtype, spare=3, heads_first=False):
    """Random pages, a table that hands them out in no order, -1 behind each sequence."""
    need = [-(-n // page_rows) for n in lengths]
    pages = sum(need) + spare
    order = list(rng.permutation(pages)[:sum(need)])
    table = np.full((len(lengths), max(need) + 1), -1, dtype=np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    host = [round_to(rng.normal(size=(pages, page_rows, hk, d)), _NAMES[dtype]) for d in (d_qk, d_v)]
    dev = [_t(x.transpose(0, 2, 1, 3), dtype).transpose(1, 2) if heads_first else _t(x, dtype) for x in host]
    return host, dev, table


@pytest.mark.parametrize("h,hk,d,dv,rotary,offset,page_rows", [
    (4, 2, 128, 128, 128, 0, 16), (2, 2, 192, 128, 64, 128, 64), (3, 1, 64, 40, 16, 8, 48),
    (2, 1, 40, 128, 24, 8, 32), (1, 1, 16, 256, 16, 0, 16)])
@pytest.mark.parametrize("new,cached", [([1], [0]), ([1, 1, 1], [15, 0, 100]), ([40, 0, 1, 17], [3, 9, 64, 0]),
                                        ([5, 5], [-2, 30])])
@pytest.mark.parametrize("heads_first", [False, True])
def test_appends_match_oracle(rng, h, hk, d, dv, rotary, offset, page_rows, new, cached, heads_first):
    """New tokens land at their positions and nothing else changes; a length below the
    new tokens' number leaves the first of them without a place."""
    from local_kimi_amd.kernels import paged_append, qk_norm_rope_append

    dtype = torch.bfloat16
    lengths = [a + b for a, b in zip(new, cached)]
    host, dev, table = _cache(rng, lengths, page_rows, hk, d, dv, dtype, heads_first=heads_first)
    rows = sum(new) + 2
    q, k, v = (round_to(rng.normal(size=(rows, n, m)), "bfloat16") for n, m in ((h, d), (hk, d), (hk, dv)))
    w = [round_to(1 + 0.3 * rng.normal(size=d), "bfloat16") for _ in range(2)]
    cs, cu = _angles(rng, 128, rotary), _cu(new)
    at = P.places(table, lengths, page_rows, host[0].shape[0], rows, cu)
    calls = {"cu_seqlens": _t(cu, torch.int32)}
    tl = (_t(table, torch.int32), _t(np.array(lengths), torch.int64))
    got = qk_norm_rope_append(_t(q[None], dtype), _t(k[None], dtype), _t(v[None], dtype), *dev, *tl,
                              _t(cs, torch.float32), *(_t(x, dtype) for x in w), 1e-6,
                              rotary_offset=offset, interleaved=heads_first, **calls)
    for x, heads, weight in ((q, None, w[0]), (k, host[0], w[1])):
        want, size = P.rotate(x, cs, at[:, 1], weight, 1e-6, offset, heads_first)
        bound = _head_bound(want, size, d, dtype)
        if heads is None:
            want[at[:, 0] < 0] = 0.0
            _close(got, want, bound, "q")
            assert not got[0, sum(new):].any()
        else:
            full, limit = heads.copy(), np.zeros_like(heads)
            for i, (_, _, page, row) in enumerate(at):
                if page >= 0:
                    full[page, row], limit[page, row] = want[i], bound[i]
            _close(dev[0], full, limit, "k")
    full = host[1].copy()
    for i, (_, _, page, row) in enumerate(at):
        if page >= 0:
            full[page, row] = v[i]
    assert np.array_equal(_np(dev[1]), full)
    # as they are
    paged_append(_t(k[None], dtype), _t(v[None], dtype), *dev, *tl, **calls)
    for full, x, t in ((host[0].copy(), k, dev[0]), (full, v, dev[1])):
        for i, (_, _, page, row) in enumerate(at):
            if page >= 0:
                full[page, row] = x[i]
        assert np.array_equal(_np(t), full)


def test_appends_write_nowhere_without_a_page(rng):
    """Tables that name no page (below 0, beyond the cache), lengths beyond the table."""
    from local_kimi_amd.kernels import paged_append

    dev = [torch.zeros((4, 16, 2, 64), device=DEV, dtype=torch.float16) for _ in range(2)]
    k = torch.ones((5, 1, 2, 64), device=DEV, dtype=torch.float16)
    table = torch.tensor([[-1, -5], [4, 2 ** 31 - 1], [-(2 ** 31), 7], [0, 1], [2, 3]], dtype=torch.int32,
                         device=DEV)
    paged_append(k, 2 * k, *dev, table, torch.tensor([3, 20, 1, 0, 2 ** 31 - 1], dtype=torch.int32, device=DEV))
    assert not dev[0].any() and not dev[1].any()
    # three tokens of which the first alone is within the table
    three = k[:1].expand(1, 3, 2, 64) * torch.arange(1, 4, device=DEV)[:, None, None].half()
    paged_append(three, three, *dev, table[3:4], torch.tensor([34], device=DEV))
    for t in dev:
        want = torch.zeros_like(t)
        want[1, 15] = 1
        assert torch.equal(t, want)


# ---------------------------------------------------------------------------
# attention


def _attend(rng, new, cached, page_rows, h, hk, dq, dv, dtype, scale=None, heads_first=False, packed=True,
            spare_rows=2):
    from local_kimi_amd.kernels import attention_paged

    lengths = [max(0, a + b) for a, b in zip(new, cached)]
    host, dev, table = _cache(rng, lengths, page_rows, hk, dq, dv, dtype, heads_first=heads_first)
    rows = sum(new) + (spare_rows if packed else 0)
    q = round_to(rng.normal(size=(rows, h, dq)), _NAMES[dtype])
    scale = dq ** -0.5 if scale is None else scale
    cu = _cu(new) if packed else None
    qt = _t(q, dtype).reshape(1 if packed else len(new), -1, h, dq)
    args = (qt, *dev, _t(table, torch.int32), _t(np.array(lengths), torch.int32))
    kw = {"scale": scale, "cu_seqlens": None if cu is None else _t(cu, torch.int32)}
    got = attention_paged(*args, **kw)
    want, spread, score, keys = P.attention_paged(q, *host, table, lengths, scale, cu)
    half = torch.finfo(dtype).eps / 2
    fp32 = 2.0 ** -24 * (2 * (dq + 8) * score[..., None] + keys + 8) * spread
    bound = half * (1 + half) * (spread + np.abs(want)) + 1.1 * fp32 + 2.0 ** -25
    _close(got, want, bound, f"{new} {cached} page {page_rows} {h}/{hk} {dq}/{dv}")
    if packed:
        assert not got[0, sum(new):].any()
    assert torch.equal(got, attention_paged(*args, **kw))
    return args, kw, got


@pytest.mark.parametrize("h,hk,dq,dv", [(4, 1, 128, 128), (32, 1, 128, 128), (2, 2, 192, 128), (6, 3, 64, 64), (2, 1, 72, 40),
                                        (1, 1, 8, 8), (32, 1, 64, 128), (10, 2, 136, 64), (7, 1, 128, 24)])
@pytest.mark.parametrize("new,cached", [([1], [0]), ([1, 1, 1, 1], [0, 63, 64, 130]), ([1, 1], [700, 3]),
                                        ([5, 0, 2], [100, 9, 0]), ([37, 1, 150], [0, 300, 45]),
                                        ([130], [65]), ([3, 6], [-3, -2])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_matches_oracle(rng, h, hk, dq, dv, new, cached, dtype):
    _attend(rng, new, cached, 16, h, hk, dq, dv, dtype)


@pytest.mark.parametrize("page_rows", [16, 32, 48, 64, 80, 128, 256, 1008])
@pytest.mark.parametrize("new,cached", [([1, 1, 1], [15, 16, 290]), ([70, 2], [101, 33])])
def test_pages_of_all_sizes_end_inside_tiles(rng, page_rows, new, cached):
    for heads_first in (False, True):
        _attend(rng, new, cached, page_rows, 4, 2, 128, 128, torch.bfloat16, heads_first=heads_first)


@pytest.mark.parametrize("b,s,cached", [(3, 1, 50), (2, 10, 200), (4, 2, 1000), (2, 70, 5)])
def test_batches_of_equal_sequences(rng, b, s, cached):
    _attend(rng, [s] * b, [cached] * b, 64, 4, 2, 64, 64, torch.float16, packed=False)


@pytest.mark.parametrize("new,cached", [([1], [3000]), ([1] * 5, [2500, 0, 70, 1, 900]), ([8], [2000]),
                                        ([1, 140, 1], [1500, 800, 2]), ([0, 1], [5, 2900])])
def test_long_caches_in_runs(rng, new, cached):
    """Keys split over blocks and joined, beside sequences that are not."""
    _attend(rng, new, cached, 16, 4, 1, 128, 128, torch.bfloat16)
    _attend(rng, new, cached, 64, 2, 2, 192, 128, torch.float16)


def test_more_sequences_than_a_wave_has_lanes(rng):
    new = [int(n) for n in rng.integers(0, 4, 150)]
    cached = [int(n) for n in rng.integers(0, 90, 150)]
    _attend(rng, new, cached, 16, 2, 1, 64, 64, torch.bfloat16)
    _attend(rng, [1] * 131, [int(n) for n in rng.integers(0, 200, 131)], 32, 2, 1, 64, 64, torch.bfloat16,
            packed=False)


@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0])
def test_sharp_negative_and_flat_scores(rng, scale):
    _attend(rng, [1, 90], [700, 20], 32, 2, 1, 128, 128, torch.bfloat16, scale=scale)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("new,cached", [([1, 3], [40, 100]), ([40, 100], [30, 3]), ([2, 1], [1300, 700])])
def test_what_a_query_does_not_see_has_no_part(rng, bad, new, cached):
    """Bad values in free pages, behind each sequence's end, and in the last positions: only
    the queries that see those may change."""
    from local_kimi_amd.kernels import attention_paged

    args, kw, clean = _attend(rng, new, cached, 16, 4, 2, 128, 64, torch.bfloat16)
    q, k, v, table, lengths = args
    k, v = k.clone(), v.clone()
    held = set()
    for s, n in enumerate(lengths.tolist()):
        for p in range(-(-n // 16)):
            page = int(table[s, p])
            held.add(page)
            for t in (k, v):
                t[page, max(0, n - 16 * p):] = bad
    for page in set(range(k.shape[0])) - held:
        k[page], v[page] = bad, bad
    assert torch.equal(attention_paged(q, k, v, table, lengths, **kw), clean)
    for back in (1, 2):  # the last positions: seen by the last queries alone
        at = 0
        k2, v2 = k.clone(), v.clone()
        for s, n in enumerate(new):
            p = int(lengths[s]) - back
            k2[int(table[s, p // 16]), p % 16] = bad
            v2[int(table[s, p // 16]), p % 16] = bad
        got = attention_paged(q, k2, v2, table, lengths, **kw)
        for n in new:
            m = max(0, n - back)
            assert torch.equal(got[0, at:at + m], clean[0, at:at + m]), (back, n)
            at += n


def test_positions_without_a_page_read_as_zeros(rng):
    from local_kimi_amd.kernels import attention_paged

    args, kw, _ = _attend(rng, [1, 40], [300, 90], 16, 4, 2, 128, 128, torch.float16)
    q, k, v, table, lengths = args
    zero = torch.zeros_like(k[:1]), torch.zeros_like(v[:1])
    k2, v2 = torch.cat((k, zero[0])), torch.cat((v, zero[1]))
    for bad in (-1, k.shape[0], 2 ** 31 - 1, -(2 ** 31)):
        named, none = table.clone(), table.clone()
        for s, b in ((0, 3), (0, 18), (1, 0), (1, 8)):
            named[s, b], none[s, b] = k.shape[0], bad
        want = attention_paged(q, k2, v2, named, lengths, **kw)
        assert torch.equal(attention_paged(q, k, v, none, lengths, **kw), want), bad


def test_graph_replays_with_other_lengths_and_pages(rng):
    """Two captured graphs in turn, eager work between the replays."""
    from local_kimi_amd.kernels import attention_paged

    dtype, n, width = torch.bfloat16, 6, 90
    k, v = (torch.randn((n * width, 16, 2, 128), device=DEV).to(dtype) for _ in range(2))
    q = torch.randn((1, 300, 8, 128), device=DEV).to(dtype)
    table = torch.zeros((n, width), dtype=torch.int32, device=DEV)
    lengths = torch.zeros(n, dtype=torch.int32, device=DEV)
    cu = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
    call = lambda: attention_paged(q, k, v, table, lengths, cu_seqlens=cu)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for new, cached in (([1] * 6, [1400, 0, 3, 700, 64, 65]), ([0] * 6, [9] * 6), ([200, 1, 1, 0, 97, 1], [0, 1300, 5, 5, 400, 2]),
                        ([300, 0, 0, 0, 0, 0], [1100, 0, 0, 0, 0, 0]), ([1] * 6, [1439] * 6)):
        table.copy_(_t(rng.permutation(n * width).reshape(n, width), torch.int32))
        lengths.copy_(_t(np.array(new) + np.array(cached), torch.int32))
        cu.copy_(_t(_cu(new), torch.int32))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = call()
        _ = (want.float() * 2).sum().item()  # unrelated eager work between replays
        for o in outs:
            assert torch.equal(o, want), new


# ---------------------------------------------------------------------------
# copies, and all of it together


@pytest.mark.parametrize("pairs", [1, 3, 192, 193, 700, 30000])
def test_copies_of_pages(rng, pairs):
    from local_kimi_amd.kernels import copy_pages

    pages = 2 * pairs + 5
    ts = [torch.randn((pages, 16, 2, 24), device=DEV).half(),
          torch.randn((pages, 2, 16, 8), device=DEV).half().transpose(1, 2),
          torch.randn((pages, 3, 40), device=DEV)[:, :, :].contiguous()[:, 1],  # every third row
          torch.randint(0, 99, (pages, 1040), device=DEV, dtype=torch.uint8)]
    want = [t.clone() for t in ts]
    order = rng.permutation(pages)
    src, dst = [int(x) for x in order[:pairs]], [int(x) for x in order[pairs:2 * pairs]]
    src[-1] = src[0]  # one page to two
    copy_pages(ts, src + [int(order[-1])], torch.tensor(dst + [int(order[-1])]))
    for t, w in zip(ts, want):
        w[dst] = w[src]
        assert torch.equal(t, w)
    copy_pages([ts[0]] * 70, [], [])
    graph, t = torch.cuda.CUDAGraph(), ts[0]  # the lists travel as arguments
    with torch.cuda.graph(graph):
        copy_pages(ts, dst, src if pairs == 1 else [int(x) for x in order[:pairs]])
    t.normal_()
    first = t.clone()
    for _ in range(3):
        t.copy_(first)
        graph.replay()
        want = first.clone()
        want[[int(x) for x in order[:pairs]]] = first[dst]
        assert torch.equal(t, want)
    many = [torch.full((2, 16), float(i), device=DEV) for i in range(70)]
    for i, t in enumerate(many):
        t[1] = -i
    copy_pages(many, [1], [0])
    assert all(bool((t == -i).all()) for i, t in enumerate(many))


def test_copies_that_depend_on_each_other_are_refused():
    from local_kimi_amd.kernels import copy_pages

    t = torch.randn((8, 16, 2, 8), device=DEV)
    want = t.clone()
    for src, dst, match in (([0, 1], [2, 2], "written twice"), ([0, 2], [2, 3], "both read"), ([0, 1], [1, 0], "both read"),
                            ([8], [1], "page 8 to 1 of a cache of 8"), ([0], [-1], "to -1"), (torch.tensor([1]), [9], "to 9"),
                            ([0] * 300, [1] * 300, "written twice")):
        with pytest.raises(ValueError, match=match):
            copy_pages([t], src, dst)
    copy_pages([t], [3, 4], [3, 4])
    assert torch.equal(t, want)


def test_a_conversation_through_the_cache(rng):
    """Prompts, single tokens, a fork that diverges, a freed sequence, a compaction: at
    each step every layer's attention equals dense attention over the same tokens, and the
    cache holds what dense rotation gives."""
    from local_kimi_amd.kernels import (attention_paged, attention_prefill, qk_norm_rope,
                                        qk_norm_rope_append, rope_table)
    from local_kimi_amd.paged import PagedCache

    layers, h, hk, d, dv, dtype = 2, 4, 2, 128, 64, torch.bfloat16
    cache = PagedCache(40, 5, 300, layers=layers, kv_heads=hk, d_qk=d, d_v=dv, page_rows=16, dtype=dtype)
    cs = rope_table(300, d, device=DEV)
    w = [(1 + 0.2 * torch.randn(d, device=DEV)).to(dtype) for _ in range(2)]
    gen = torch.Generator(device=DEV).manual_seed(3)
    dense = {}  # sequence -> per layer (k, v) of all its tokens, rotated

    def step(seqs, counts):
        cache.extend(seqs, counts)
        table, lengths = cache.rows_of(seqs)
        cu = _t(_cu(counts), torch.int32)
        for layer in range(layers):
            q, k, v = (torch.randn((1, sum(counts), n, m), generator=gen, device=DEV).to(dtype)
                       for n, m in ((h, d), (hk, d), (hk, dv)))
            pages = cache.k_pages[layer], cache.v_pages[layer]
            qr = qk_norm_rope_append(q, k, v, *pages, table, lengths, cs, *w, 1e-6, cu_seqlens=cu)
            got = attention_paged(qr, *pages, table, lengths, cu_seqlens=cu)
            at = 0
            for s, n in zip(seqs, counts):
                had = dense[s][layer][0].shape[1] if dense[s][layer] else 0
                pos = torch.arange(had, had + n, device=DEV)[None]
                q1, k1 = qk_norm_rope(q[:, at:at + n], k[:, at:at + n], cs, pos, *w, 1e-6)
                assert torch.equal(q1, qr[:, at:at + n])
                old = dense[s][layer] or (k1[:, :0], v[:, :0])
                new = torch.cat((old[0], k1), 1), torch.cat((old[1], v[:, at:at + n]), 1)
                dense[s][layer] = new
                want = attention_prefill(q1, *new)
                # both round p and the output once, each off by eps / 2 of sum p |v| <= max |v|, twice
                near = 4 * torch.finfo(dtype).eps / 2 * new[1].float().abs().amax()
                assert bool(((got[:, at:at + n].float() - want.float()).abs() <= near).all())
                used = table[seqs.index(s), :-(-(had + n) // 16)].long()
                assert torch.equal(pages[0][used].flatten(0, 1)[:had + n], new[0][0])
                assert torch.equal(pages[1][used].flatten(0, 1)[:had + n], new[1][0])
                at += n

    a, b = cache.add(), cache.add()
    dense[a], dense[b] = [None] * layers, [None] * layers
    step([a, b], [37, 90])
    for _ in range(3):
        step([b, a], [1, 1])
    c = cache.fork(a)
    dense[c] = list(dense[a])
    step([a, b, c], [1, 1, 1])  # a's and c's last page parts here
    step([c, a], [30, 2])
    before = cache.book.free_pages
    cache.free(b)
    assert cache.book.free_pages > before
    assert cache.compact() > 0
    step([a, c], [1, 5])
    d2 = cache.fork(c)
    dense[d2] = list(dense[c])
    step([d2, c, a], [3, 1, 1])
    # all sequences of the cache at once, those not in use among them
    seqs = [a, b, c, d2, 4]
    cache.extend([a, c, d2], [1, 1, 1])
    q = torch.randn((5, 1, h, d), device=DEV).to(dtype)
    out = attention_paged(q, cache.k_pages[0], cache.v_pages[0], cache.page_table, cache.lengths)
    unused = [s for s in range(5) if cache.book.pages[s] is None]
    assert len(unused) == 2 and not out[unused].any() and out[[a, c, d2]].any(), seqs
