"""What the paged-cache operators promise beyond their sums: results do not depend on
what a query does not see nor on where the pages lie, caches beyond 4 GB, other streams,
captured decode steps, layouts, and tables or offsets that lead nowhere.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .test_gpu_paged import DEV, _attend, _cu, _require_gpu, _t

pytestmark = pytest.mark.gpu

_ = _require_gpu  # fixture


def _case(seed, new, cached, page_rows=16, h=8, hk=2, dq=128, dv=128, dtype=torch.bfloat16, spare=4):
    """q, pages, table, lengths, offsets of random packed sequences on the device."""
    rng = np.random.default_rng(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    lengths = [a + b for a, b in zip(new, cached)]
    need = [-(-n // page_rows) for n in lengths]
    order = rng.permutation(sum(need) + spare)[:sum(need)]
    table, at = np.full((len(new), max(need) + 1), -1, dtype=np.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    q, k, v = (torch.randn(s, generator=g, device=DEV).to(dtype)
               for s in ((1, sum(new), h, dq), (sum(need) + spare, page_rows, hk, dq),
                         (sum(need) + spare, page_rows, hk, dv)))
    return q, k, v, _t(table, torch.int32), _t(np.array(lengths), torch.int32), _t(_cu(new), torch.int32)


def _at(table, s, p, page_rows=16):
    return int(table[s, p // page_rows]), p % page_rows


@pytest.mark.parametrize("new,cached", [([3, 2], [90, 700]), ([150], [200]), ([8], [2000]), ([1, 40], [1500, 800])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_later_finite_keys_change_nothing(new, cached, dtype):
    """The last position's key, large enough to be the maximum of the query that sees it
    by far: the earlier queries' results stay bit for bit."""
    from local_kimi_amd.kernels import attention_paged

    for seed in range(6):
        q, k, v, table, lengths, cu = _case(seed, new, cached, dtype=dtype)
        clean = attention_paged(q, k, v, table, lengths, cu_seqlens=cu, scale=0.2)
        k = k.clone()
        at = 0
        for s, n in enumerate(new):
            page, row = _at(table, s, int(lengths[s]) - 1)
            k[page, row] = 8 * q[0, at + n - 1, ::4]
            at += n
        got = attention_paged(q, k, v, table, lengths, cu_seqlens=cu, scale=0.2)
        at = 0
        for n in new:
            assert torch.equal(got[0, at:at + n - 1], clean[0, at:at + n - 1])
            assert not torch.equal(got[0, at + n - 1], clean[0, at + n - 1])
            at += n


@pytest.mark.parametrize("new,cached", [([4], [400]), ([20], [400]), ([1], [3000])])
def test_another_heads_queries_change_nothing(new, cached):
    from local_kimi_amd.kernels import attention_paged

    q, k, v, table, lengths, cu = _case(1, new, cached)
    clean = attention_paged(q, k, v, table, lengths, cu_seqlens=cu, scale=0.2)
    q = q.clone()
    q[:, :, 1::4] *= 8
    got = attention_paged(q, k, v, table, lengths, cu_seqlens=cu, scale=0.2)
    for head in (0, 2, 3, 4, 6, 7):
        assert torch.equal(got[:, :, head], clean[:, :, head])


@pytest.mark.parametrize("new,cached", [([1, 1, 1], [900, 5, 300]), ([70, 1], [333, 1200])])
def test_where_pages_lie_changes_nothing(new, cached):
    """Other pages, pages of another size, of heads first, sequences that share theirs."""
    from local_kimi_amd.kernels import attention_paged

    q, k, v, table, lengths, cu = _case(2, new, cached)
    want = attention_paged(q, k, v, table, lengths, cu_seqlens=cu)
    order = torch.randperm(k.shape[0], device=DEV)
    moved = torch.where(table >= 0, torch.argsort(order).int()[table.clamp(min=0).long()], -1)
    assert torch.equal(attention_paged(q, k[order], v[order], moved, lengths, cu_seqlens=cu), want)
    first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    assert torch.equal(attention_paged(q, *first, table, lengths, cu_seqlens=cu), want)
    one = torch.stack((torch.cat((k, k), -1), torch.cat((v, v), -1)), 1)[..., 128:]  # side by side
    assert torch.equal(attention_paged(q, one[:, 0], one[:, 1], table, lengths, cu_seqlens=cu), want)
    # pairs of pages as one of twice the rows
    wide = [torch.cat((t[table.clamp(min=0).long()].flatten(1, 2),
                       torch.zeros_like(t[table.clamp(min=0).long()].flatten(1, 2))[:, :48]), 1) for t in (k, v)]
    rows = wide[0].shape[1] // 48 * 48
    wide = [t[:, :rows].reshape(-1, 48, *t.shape[2:]) for t in wide]
    named = torch.arange(wide[0].shape[0], device=DEV, dtype=torch.int32).reshape(len(new), -1)
    assert torch.equal(attention_paged(q, *wide, named, lengths, cu_seqlens=cu), want)


def test_layouts_of_queries_tables_and_lengths():
    from local_kimi_amd.kernels import attention_paged

    q, k, v, table, lengths, _ = _case(3, [2, 2, 2], [50, 0, 333])
    q = q.reshape(3, 2, 8, 128)
    want = attention_paged(q, k, v, table, lengths)
    fused = torch.zeros((3, 2, 8, 136), device=DEV).bfloat16()
    odd = torch.zeros((3, 2, 8, 129), device=DEV).bfloat16()
    for t in (fused[..., :128], odd[..., 1:], torch.zeros((2, 3, 8, 128), device=DEV).bfloat16().transpose(0, 1)):
        t.copy_(q)
        assert torch.equal(attention_paged(t, k, v, table, lengths), want)
    wide = torch.full((3, 99), 7, dtype=torch.int32, device=DEV)
    wide[:, 5:5 + table.shape[1]] = table
    for t in (wide[:, 5:5 + table.shape[1]], table.t().contiguous().t()):
        assert torch.equal(attention_paged(q, k, v, t, lengths.long()), want)
    assert torch.equal(attention_paged(q, k, v, table, torch.stack((lengths, lengths), 1)[:, 0]), want)
    last = torch.zeros((3, 5, 8, 128), device=DEV).bfloat16()
    last[:, -1:] = q[:, 1:]
    one = attention_paged(q[:, 1:].contiguous(), k, v, table, lengths)
    assert torch.equal(attention_paged(last[:, -1:], k, v, table, lengths), one)
    # one row of the table for all
    same = attention_paged(q, k, v, table[:1].expand(3, -1), lengths[:1].expand(3))
    assert torch.equal(same, attention_paged(q, k, v, table[:1].repeat(3, 1), lengths[:1].repeat(3)))


def test_calls_without_rows_pages_or_keys():
    from local_kimi_amd.kernels import attention_paged, paged_append, qk_norm_rope_append

    q, k, v, table, lengths, cu = _case(4, [2, 3], [20, 30])
    assert attention_paged(q[:, :0], k, v, table, lengths, cu_seqlens=0 * cu).shape == (1, 0, 8, 128)
    for t, kk, vv in ((table[:, :0], k, v), (table, k[:0], v[:0]), (torch.full_like(table, -1), k, v)):
        got = attention_paged(q, kk, vv, t, lengths, cu_seqlens=cu)
        assert not got.any()  # positions without a page: values of zero
        before = k.clone()
        paged_append(q[:, :, :2], q[:, :, :2], kk, vv, t, lengths, cu_seqlens=cu)
        assert torch.equal(k, before)
    assert not attention_paged(q, k, v, table, 0 * lengths - 5, cu_seqlens=cu).any()
    out = qk_norm_rope_append(q, q[:, :, :2], q[:, :, :2], k[:0], v[:0], table, lengths,
                              torch.ones((9, 128), device=DEV), cu_seqlens=0 * cu)
    assert not out.any()  # every row is behind the last sequence


def test_caches_beyond_4_gb():
    """Pages whose offsets pass 2^32 bytes and elements: written, read and copied."""
    from local_kimi_amd.kernels import attention_paged, copy_pages, paged_append

    rows, hk, d = 64, 8, 128
    pages = (1 << 32) // (rows * hk * d) + 40  # 4.3e9 elements, 8.6 GB
    k = torch.empty((pages, rows, hk, d), dtype=torch.bfloat16, device=DEV)
    low = torch.randn((12, rows, hk, d), device=DEV).bfloat16()
    lengths = torch.tensor([200, 300], dtype=torch.int32, device=DEV)
    small = torch.arange(10, dtype=torch.int32, device=DEV).reshape(2, 5)
    high = small + (pages - 12)
    new = torch.randn((2, 130, hk, d), device=DEV).bfloat16()
    q = torch.randn((2, 130, 32, d), device=DEV).bfloat16()
    v, low_v = torch.empty_like(k), low.flip(0)
    k[pages - 12:], v[pages - 12:] = low, low_v
    for pair, table in (((low, low_v), small), ((k, v), high)):
        paged_append(new, 2 * new, *pair, table, lengths)
    assert torch.equal(k[pages - 12:], low) and torch.equal(v[pages - 12:], low_v)
    for n in (1, 130):
        want = attention_paged(q[:, :n], low, low_v, small, lengths)
        assert torch.equal(attention_paged(q[:, :n], k, v, high, lengths), want)
    k[1] = 0
    copy_pages([k], [pages - 3, 1], [0, pages - 1])
    assert torch.equal(k[0], low[9]) and not k[pages - 1].any()


def test_another_stream_and_two_calls_at_once():
    from local_kimi_amd.kernels import attention_paged

    cases = [_case(s, [1] * 20, [int(x) for x in np.random.default_rng(s).integers(0, 3000, 20)]) for s in (5, 6)]
    want = [attention_paged(*c[:5], cu_seqlens=c[5]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for i, (stream, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(stream):
                got[i].append(attention_paged(*c[:5], cu_seqlens=c[5]))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)


def test_a_captured_decode_step_follows_its_lengths():
    """lengths += 1, append and attention in one graph: replays are the eager steps. A
    sequence that is not in use stays out."""
    from local_kimi_amd.kernels import attention_paged, qk_norm_rope_append, rope_table

    n, width, h, hk, d, dtype = 5, 40, 8, 2, 128, torch.bfloat16
    cs = rope_table(16 * width, d, device=DEV)
    table = torch.randperm(n * width, device=DEV).int().reshape(n, width)
    start = torch.tensor([0, 15, 16, 500, 0], dtype=torch.int32, device=DEV)
    used = torch.tensor([1, 1, 1, 1, 0], dtype=torch.int32, device=DEV)
    x = torch.randn((12, n, 1, h + 2 * hk, d), device=DEV).to(dtype)
    first = [torch.randn((n * width, 16, hk, d), device=DEV).to(dtype) for _ in range(2)]
    w = torch.ones(d, device=DEV)

    def step(inp, k, v, lengths):
        lengths += used
        q = qk_norm_rope_append(inp[:, :, :h], inp[:, :, h:h + hk], inp[:, :, h + hk:], k, v, table, lengths, cs, w, w)
        return attention_paged(q, k, v, table, lengths)

    eager = [t.clone() for t in first], start.clone()
    want = [step(x[i], *eager[0], eager[1]) for i in range(12)]
    static, state = x[0].clone(), ([t.clone() for t in first], start.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static, *state[0], state[1])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static, *state[0], state[1])
    for t, f in zip(state[0], first):
        t.copy_(f)
    state[1].copy_(start)
    for i in range(12):
        static.copy_(x[i])
        graph.replay()
        assert torch.equal(out, want[i]), i
        assert not out[4].any()
        _ = (out.float() + 1).sum().item()  # unrelated work between replays
    for a, b in zip(state[0], eager[0]):
        assert torch.equal(a, b)


def test_a_cache_that_is_extended_while_its_steps_run():
    """Uploads take their turn on the stream: 30 steps issued without a wait equal the
    same steps one by one."""
    from local_kimi_amd.kernels import attention_paged, paged_append
    from local_kimi_amd.paged import PagedCache

    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn((30, 4, 1, 2, 128), generator=g, device=DEV).bfloat16()
    outs = []
    for wait in (True, False):
        cache = PagedCache(64, 6, 200, layers=1, kv_heads=2, d_qk=128, d_v=128, page_rows=16)
        seqs = [cache.add() for _ in range(3)]
        cache.extend(seqs, [100, 14, 31])
        got = []
        for i in range(30):
            if i == 10:
                seqs.append(cache.fork(seqs[2]))
            cache.extend(seqs, [1] * len(seqs))
            if wait:
                torch.cuda.synchronize()
            n = len(seqs)
            table, lengths = cache.rows_of(seqs)
            paged_append(x[i, :n], x[i, :n], cache.k_pages[0], cache.v_pages[0], table, lengths)
            got.append(attention_paged(x[i, :n], cache.k_pages[0], cache.v_pages[0], table, lengths))
        outs.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("cu", [[0, 90, 30, 60, 100], [40, 20, 0, 300, 100], [-7, 5, 2 ** 31 - 1, 3, 9], [100, 100, 0, 0, 0],
                                [0, 0, 0, 0, -5]])
def test_offsets_out_of_order_lead_nowhere(cu):
    """Results within such calls are left open; what is not theirs stays as it was."""
    from local_kimi_amd.kernels import attention_paged, paged_append

    q, k, v, table, lengths, _ = _case(7, [25] * 4, [700, 3, 1200, 60])
    bad = torch.tensor(cu, dtype=torch.int32, device=DEV)
    assert attention_paged(q, k, v, table, lengths, cu_seqlens=bad).shape == (1, 100, 8, 128)
    free = sorted(set(range(k.shape[0])) - set(table.flatten().tolist()))
    before = k.clone()
    paged_append(q[:, :, :2], q[:, :, :2], k, v, table, lengths, cu_seqlens=bad)
    assert torch.equal(k[free], before[free])
    torch.cuda.synchronize()


@pytest.mark.parametrize("keys", [41, 1500])
def test_largest_fp16_values_stay_finite(keys):
    """Means of +-65504 under weights that fp16 rounds up (as for dense keys)."""
    from local_kimi_amd.kernels import attention_paged

    pages = -(-keys // 16)
    q = torch.zeros((1, 3, 1, 64), device=DEV, dtype=torch.float16)
    q[..., 0] = 1
    k = torch.zeros((pages, 16, 1, 64), device=DEV, dtype=torch.float16)
    k.view(-1, 64)[1:, 0] = -1
    v = torch.full_like(k, 65504.0)
    v[..., 1::2] = -65504.0
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    lengths = torch.tensor([keys], dtype=torch.int32, device=DEV)
    scale = -float(np.log(0.5 + 1.1 * 2.0 ** -12))
    got = attention_paged(q, k, v, table, lengths, scale=scale)
    assert torch.equal(got, v.view(1, -1, 1, 64)[:, :3])
    v.view(-1, 64)[0, 3] = float("inf")
    got = attention_paged(q, k, v, table, lengths, scale=scale)
    assert bool((got[..., 3] == float("inf")).all()) and torch.equal(got[..., 4:], v.view(1, -1, 1, 64)[:, 4:7, :, 4:])


@pytest.mark.parametrize("keys", [150, 2500])
@pytest.mark.parametrize("rows", [1, 40])
def test_scores_of_minus_infinity(rng, keys, rows):
    """Keys whose score is -infinity have no weight; a query that sees no other gets zeros."""
    from local_kimi_amd.kernels import attention_paged

    args, kw, clean = _attend(rng, [rows], [keys], 16, 2, 1, 64, 64, torch.bfloat16)
    q, k, v, table, lengths = args
    q, k = q.clone(), k.clone()
    q[..., 0] = 1.0
    k[..., 0] = -float("inf")
    assert not attention_paged(q, k, v, table, lengths, **kw).any()
    k[int(table[0, 2])] = 0.0  # sixteen keys of one score: the mean of their values
    got = attention_paged(q, k, v, table, lengths, **kw)[0, :rows, 0].float()
    mean = v[int(table[0, 2]), :, 0].float().mean(0)
    # p of one, sums of sixteen: one rounding of the result
    assert bool(((got - mean).abs() <= 2.0 ** -8 * mean.abs() + 2.0 ** -20).all())


@pytest.mark.parametrize("n", [255, 256, 700, 1500])
def test_many_sequences_in_all_forms(n):
    """Around and beyond the number from which a launch of its own counts them: each
    sequence alone gives its results to a rounding of each side's p and sums."""
    from local_kimi_amd.kernels import attention_paged

    rng = np.random.default_rng(n)
    new = [int(x) for x in rng.integers(0, 3, n)]
    cached = [int(x) for x in rng.integers(0, 40, n)]
    new[7], cached[7] = 40, 30
    new[n - 3], cached[n - 3] = 1, 5000
    new[n // 2], cached[n // 2] = 5, 2000
    q, k, v, table, lengths, cu = _case(n, new, cached, h=4, hk=2, dq=64, dv=64)
    q = torch.cat((q, torch.ones_like(q[:, :70])), 1)  # rows behind the last sequence
    got = attention_paged(q, k, v, table, lengths, cu_seqlens=cu)
    assert torch.equal(got, attention_paged(q, k, v, table, lengths, cu_seqlens=cu))
    assert not got[0, sum(new):].any()
    at, largest = np.concatenate(([0], np.cumsum(new))), v.float().abs().amax().item()
    for s in sorted({*range(0, n, 29), 7, n // 2, n - 3, n - 1}):
        if new[s]:
            rows = slice(int(at[s]), int(at[s + 1]))
            one = attention_paged(q[:, rows], k, v, table[s:s + 1], lengths[s:s + 1])
            # p and the output rounded on both sides, each by 2^-9 of at most the largest value
            assert (got[:, rows].float() - one.float()).abs().amax().item() <= 4 * 2.0 ** -9 * largest, s
    # a batch of single tokens, none in runs
    q1 = torch.randn((n, 1, 4, 64), device=DEV).bfloat16()
    few = lengths.clamp(max=100)
    got = attention_paged(q1, k, v, table[:, :8], few)
    one = torch.cat([attention_paged(q1[i:i + 1], k, v, table[i:i + 1, :8], few[i:i + 1]) for i in range(0, n, 50)])
    assert torch.equal(got[::50], one)
