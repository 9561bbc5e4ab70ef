"""GPU parity of the prompt kernels at the ends of their ranges: many sequences,
many and wide heads, workspaces of several windows, offsets beyond 32 bits, runs
of the keys, values that must not reach other queries.

Tolerances as in test_gpu_kda_prefill.py and test_gpu_attention.py, whose checks
these tests call; where two calls compute the same sums in the same order,
their results are equal bit by bit.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kda as K

from .test_gpu_attention import _check, _inputs
from .test_gpu_kda_prefill import (DEV, _close, _conv_check, _conv_inputs, _cu, _np, _require_gpu,
                                   _run_scan, _scan_inputs, _scan_tol, _t, form)

pytestmark = pytest.mark.gpu

_ = _require_gpu, form  # fixtures


def _ragged(rng, n, longest):
    """n lengths from 0 to longest, some of them empty, none of them all."""
    lengths = rng.integers(0, longest + 1, size=n)
    lengths[::7] = 0
    lengths[n // 2] = longest
    return lengths.tolist()


@pytest.mark.parametrize("n,longest", [(63, 5), (64, 20), (100, 40), (5000, 2)])
def test_many_sequences(rng, form, n, longest):
    from local_kimi_amd.kernels import attention_prefill, short_conv_prefill_triple

    lengths = _ragged(rng, n, longest)
    cu, rows = _cu(lengths), sum(lengths) + 2
    a = _scan_inputs(rng, rows, 1, 8, 12, n)
    want_state, want = K.prefill(*a, 0.5, cu)
    out, st = _run_scan(a, cu, torch.float32, 0.5)
    _close(out, want, longest, torch.float32, "scan")
    _close(st, want_state, longest, torch.float32, "states")
    assert not out[sum(lengths):].any()

    x, s, w = _conv_inputs(rng, rows, n, 8, torch.bfloat16)
    states = [_t(t, torch.bfloat16) for t in s]
    outs = short_conv_prefill_triple(*(_t(t[None], torch.bfloat16) for t in x), *states,
                                     *(_t(t, torch.bfloat16) for t in w), cu_seqlens=_t(cu, torch.int32))
    for i in range(3):
        _conv_check(outs[i][0], x[i], s[i], w[i], torch.bfloat16, cu, f"conv {i}")
        assert np.array_equal(_np(states[i]), K.short_conv_prefill(x[i], s[i], w[i], "float32", cu)[1])

    keys = [n + int(extra) for n, extra in zip(lengths, rng.integers(0, 4, size=n))]
    b = _inputs(rng, rows, sum(keys) + 1, 2, 1, 64, 64, torch.bfloat16)
    cuk = _cu(keys)
    got = attention_prefill(*(_t(t[None], torch.bfloat16) for t in b), scale=0.1,
                            cu_seqlens=_t(cu, torch.int32), cu_seqlens_k=_t(cuk, torch.int32))
    _check(got, b, 0.1, torch.bfloat16, n, cu, cuk, "attention")
    assert not got[0, sum(lengths):].any()


@pytest.mark.parametrize("lengths,h,dk,dv", [
    ([70, 33], 2, 64, 200), ([45], 1, 128, 272),       # more value columns than a pass solves
    ([40] * 15 + [0, 65], 8, 128, 117),                # two column tiles a block: 17 x 8 x 8
    ([33, 1, 0] * 12, 6, 64, 72)])                     # and an odd number of them: 36 x 6 x 5
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_chunks_of_wide_and_many_heads(rng, lengths, h, dk, dv, dtype):
    from local_kimi_amd import _lib

    cu, rows = _cu(lengths), sum(lengths) + 3
    a = _scan_inputs(rng, rows, h, dk, dv, len(lengths), dtype)
    want_state, want = K.prefill(*a, dk ** -0.5, cu)
    with _lib.forced_path("kda_prefill", "chunks"):
        out, st = _run_scan(a, cu, dtype, dk ** -0.5)
    _close(out, want, max(lengths), dtype, "out")
    _close(st, want_state, max(lengths), torch.float32, "state")
    assert not out[sum(lengths):].any()


def test_windows_join(rng):
    """Records of more than one window, sequences that begin, end and go on
    across its edge: each form is within its tolerance of the exact result, so
    they are within twice that of each other."""
    from local_kimi_amd import _lib

    lengths = [3000, 0, 900, 1700, 40]
    cu, h, d = _cu(lengths), 32, 128
    need = _lib.query("lk_kda_prefill_workspace", len(lengths), sum(lengths), h, d, d)
    more = _lib.query("lk_kda_prefill_workspace", len(lengths), 10 * sum(lengths), h, d, d)
    assert need == more > 0  # a window's
    a = _scan_inputs(rng, sum(lengths), h, d, d, len(lengths), rate=0.02)
    got = {}
    for form in ("steps", "chunks"):
        with _lib.forced_path("kda_prefill", form):
            got[form] = _run_scan(a, cu, torch.float32, d ** -0.5)
    for x, y in zip(got["steps"], got["chunks"]):
        x, y = x.double(), y.double()
        tol, rms = 2 * _scan_tol(max(lengths)), float(x.square().mean().sqrt())
        assert float((x - y).square().mean().sqrt()) <= tol * rms
        assert bool(((x - y).abs() <= 8 * tol * x.abs().clamp(min=rms)).all())


@pytest.mark.parametrize("value", [float("nan"), float("inf"), 1e30])
@pytest.mark.parametrize("which", [1, 2, 3, 5])  # q, k, v, beta
def test_scan_steps_before_a_bad_one_are_untouched(rng, form, which, value):
    lengths = [100, 70]
    a = _scan_inputs(rng, 170, 2, 64, 48, 2)
    clean, _ = _run_scan(a, _cu(lengths), torch.float32, 1.0)
    for spot in (0, 15, 16, 31, 32, 47, 77):
        bad = [x.copy() for x in a]
        bad[which][spot] = value
        out, st = _run_scan(bad, _cu(lengths), torch.float32, 1.0)
        assert torch.equal(out[:spot], clean[:spot]), spot
        assert torch.equal(out[100:], clean[100:]) and torch.isfinite(st[1]).all(), spot


@pytest.mark.parametrize("h,hk", [(3, 1), (10, 2), (7, 1), (12, 1), (17, 1), (24, 1), (32, 1), (66, 2)])
def test_attention_groups(rng, h, hk):
    """Group sizes that a block's rows hold whole, in part, or one head at a time."""
    from local_kimi_amd.kernels import attention_prefill

    lq, lk = [5, 0, 47, 1], [5, 3, 50, 900]
    dtype = torch.bfloat16
    a = _inputs(rng, sum(lq) + 1, sum(lk), h, hk, 64, 40, dtype)
    got = attention_prefill(*(_t(x[None], dtype) for x in a), cu_seqlens=_t(_cu(lq), torch.int32),
                            cu_seqlens_k=_t(_cu(lk), torch.int32))
    _check(got, a, 64 ** -0.5, dtype, len(lq), _cu(lq), _cu(lk), f"{h}/{hk}")
    assert not got[0, sum(lq):].any()


@pytest.mark.parametrize("h,hk,dq,dv", [(2, 2, 192, 128), (4, 1, 64, 64)])
@pytest.mark.parametrize("lq,lk", [(1, 5000), (40, 2600), (200, 1801)])
def test_attention_in_runs_of_the_keys(rng, h, hk, dq, dv, lq, lk):
    """Few queries, many keys; bad values in keys that later queries see alone."""
    from local_kimi_amd import _lib
    from local_kimi_amd.kernels import attention_prefill

    dtype = torch.float16
    assert _lib.query("lk_attention_prefill_workspace", lq, lk, 1, h, hk, dq, dv) > 0
    a = _inputs(rng, lq, lk, h, hk, dq, dv, dtype)
    t = [_t(x[None], dtype) for x in a]
    clean = attention_prefill(*t)
    _check(clean, a, dq ** -0.5, dtype, what=f"{lq} {lk}")
    assert torch.equal(attention_prefill(*t), clean)
    for value in (float("nan"), float("inf")):
        for back in {1, lq // 2, lq - 1} - {0}:  # seen by the last `back` queries
            k, v = t[1].clone(), t[2].clone()
            k[:, lk - back], v[:, lk - back] = value, value
            got = attention_prefill(t[0], k, v)
            assert torch.equal(got[:, :lq - back], clean[:, :lq - back])
            assert not torch.isfinite(got[:, lq - back:]).any()


def test_rows_far_apart(rng):
    """Row offsets beyond 2^31 elements: the same results as from dense rows."""
    from local_kimi_amd.kernels import attention_prefill, short_conv_prefill_triple

    rows, stride = 600, 1 << 22
    wide = torch.empty((1, rows, stride), device=DEV, dtype=torch.bfloat16)  # 5 GB, most of it unused
    dense = torch.randn((1, rows, 4, 64 + 64 + 64), device=DEV).to(torch.bfloat16)
    far = wide[:, :, :dense[0, 0].numel()].view(1, rows, 4, 192)
    far.copy_(dense)
    assert far.stride(1) == stride and (rows - 1) * stride > 1 << 31
    cu = torch.tensor([0, 30, 590, rows], dtype=torch.int32, device=DEV)
    parts = [t.split(64, dim=-1) for t in (far, dense)]
    assert torch.equal(attention_prefill(*parts[0], cu_seqlens=cu),
                       attention_prefill(*(t.contiguous() for t in parts[1]), cu_seqlens=cu))
    w = [torch.randn((256, 1, 4), device=DEV).to(torch.bfloat16) for _ in range(3)]
    got = []
    for rows_of in (far, dense):
        flat = rows_of[:, :, :, :].flatten(2)
        states = [torch.zeros((3, 256, 4), device=DEV, dtype=torch.bfloat16) for _ in range(3)]
        got.append([*short_conv_prefill_triple(*flat.split(256, dim=-1), *states, *w, cu_seqlens=cu),
                    *states])
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_scan_of_more_than_2_to_the_31_values(form):
    """The last sequence of a call whose offsets pass 32 bits, against a call of
    its own."""
    from local_kimi_amd.kernels import kda_prefill

    n, length, h, dk, dv = 1100, 64, 256, 128, 16
    rows = n * length
    assert rows * h * dk > 1 << 31
    g = torch.Generator(device=DEV).manual_seed(7)
    q, k, decay = (torch.empty((1, rows, h, dk), device=DEV).uniform_(-s, s, generator=g)
                   for s in (0.1, 0.1, 0.3))
    decay.abs_().neg_()
    v = torch.empty((1, rows, h, dv), device=DEV, dtype=torch.bfloat16).uniform_(-1, 1, generator=g)
    beta = torch.empty((1, rows, h), device=DEV).uniform_(0, 1, generator=g)
    state = torch.zeros((n, h, dk, dv), device=DEV)
    cu = torch.arange(0, rows + 1, length, device=DEV)
    out = kda_prefill(state, q, k, v, decay, beta, scale=0.1, cu_seqlens=cu)
    own = torch.zeros((1, h, dk, dv), device=DEV)
    last = kda_prefill(own, *(t[:, -length:] for t in (q, k, v, decay, beta)), scale=0.1)
    assert last.abs().max() > 0
    assert torch.equal(out[:, -length:], last) and torch.equal(state[-1:], own)


def test_offsets_from_elsewhere_and_beyond_32_bits(rng, form):
    """Sequences that do not start at row 0 (rows before them are no one's), ends
    that no int32 holds."""
    from local_kimi_amd.kernels import attention_prefill, kda_prefill, short_conv_prefill_triple

    rows, first = 150, 71
    cu = np.array([first, 110, 2 ** 33 + 5])
    offsets = torch.from_numpy(cu).to(DEV)
    x, s, w = _conv_inputs(rng, rows, 2, 16, torch.bfloat16)
    states = [_t(t, torch.bfloat16) for t in s]
    outs = short_conv_prefill_triple(*(_t(t[None], torch.bfloat16) for t in x), *states,
                                     *(_t(t, torch.bfloat16) for t in w), cu_seqlens=offsets)
    for i in range(3):
        y, new = K.short_conv_prefill(x[i], s[i], w[i], "float32", cu)
        _conv_check(torch.cat((torch.zeros_like(outs[i][0, :first]), outs[i][0, first:])), x[i], s[i],
                    w[i], torch.bfloat16, cu, f"conv {i}")
        assert np.array_equal(_np(states[i]), new)
    a = _scan_inputs(rng, rows, 1, 32, 16, 2)
    want_state, want = K.prefill(*a, 1.0, cu)
    st = _t(a[0])
    out = kda_prefill(st, *(_t(t[None]) for t in a[1:]), scale=1.0, cu_seqlens=offsets)
    _close(out[0, first:], want[first:], 50, torch.float32, "scan")
    _close(st, want_state, 50, torch.float32, "states")
    b = _inputs(rng, rows, rows, 2, 1, 64, 64, torch.bfloat16)
    got = attention_prefill(*(_t(t[None], torch.bfloat16) for t in b), cu_seqlens=offsets)
    got = torch.cat((torch.zeros_like(got[:, :first]), got[:, first:]), dim=1)
    _check(got, b, 0.125, torch.bfloat16, 2, cu, cu, "attention")


def test_conv_and_attention_on_another_stream(rng):
    """Inputs made on the stream that the call runs on, while the default one is idle."""
    from local_kimi_amd.kernels import attention_prefill, short_conv_prefill_triple

    x = torch.randn((1, 900, 4, 64), device=DEV).to(torch.bfloat16)
    w = [torch.randn((256, 4), device=DEV).to(torch.bfloat16) for _ in range(3)]

    def run():
        y = (x * 0.5).contiguous()
        states = [torch.zeros((1, 256, 4), device=DEV, dtype=torch.bfloat16) for _ in range(3)]
        outs = short_conv_prefill_triple(*[y.view(1, 900, 256)] * 3, *states, *w)
        return [attention_prefill(*(t.view(1, 900, 4, 64) for t in outs)), *states]

    want = run()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = run()
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_no_tokens_and_no_keys(rng):
    """Calls without a row: states are kept (or handed on), queries without keys get zeros."""
    from local_kimi_amd.kernels import attention_prefill, kda_prefill, short_conv_prefill_triple

    def made(*shape, dtype=torch.float32):
        return _t(rng.normal(size=shape), dtype)

    state, new = made(2, 3, 16, 8), torch.zeros((2, 3, 16, 8), device=DEV)
    kept = state.clone()
    none = [torch.zeros((2, 0, 3, w), device=DEV) for w in (16, 16, 8, 16)]
    out = kda_prefill(state, *none, torch.zeros((2, 0, 3), device=DEV), scale=1.0, state_out=new)
    assert out.shape == (2, 0, 3, 8) and torch.equal(state, kept) and torch.equal(new, kept)

    states = [made(2, 24, 4, dtype=torch.float16) for _ in range(3)]
    before = [s.clone() for s in states]
    x = torch.zeros((2, 0, 24), device=DEV, dtype=torch.float16)
    w = [made(24, 4, dtype=torch.float16) for _ in range(3)]
    outs = short_conv_prefill_triple(x, x, x, *states, *w)
    assert all(o.shape == x.shape for o in outs)
    assert all(torch.equal(a, b) for a, b in zip(states, before))

    q, kv = made(2, 5, 4, 64, dtype=torch.float16), torch.zeros((2, 0, 2, 64), device=DEV, dtype=torch.float16)
    assert not attention_prefill(q, kv, kv).any()
    assert attention_prefill(q[:, :0], kv, kv).shape == (2, 0, 4, 64)


def test_graph_of_runs_and_windows_replays(rng):
    """A prompt of several windows and a query in runs of the keys, captured
    together; replayed on other values between eager work."""
    from local_kimi_amd.kernels import attention_prefill, kda_prefill

    a = [_t(x) for x in _scan_inputs(rng, 5000, 32, 128, 128, 1, rate=0.02)]
    state, args = a[0], [x[None] for x in a[1:]]
    q = _t(rng.normal(size=(1, 3, 8, 128)), torch.bfloat16)
    k, v = (_t(rng.normal(size=(1, 4000, 2, 128)), torch.bfloat16) for _ in range(2))
    start = state.clone()

    def run():
        return kda_prefill(state, *args, scale=0.1), attention_prefill(q, k, v)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for i in range(3):
        for t in (q, k, args[2]):
            t.mul_(0.75)
        state.copy_(start)
        want = [t.clone() for t in run()] + [state.clone()]
        for t in got:
            t.zero_()
        state.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip([*got, state], want):
            assert torch.equal(x, y), i


def test_two_calls_at_once(rng, form):
    """Each of two streams has a workspace of its own."""
    from local_kimi_amd.kernels import attention_prefill, kda_prefill

    calls = []
    for n in (700, 900):
        a = [_t(x) for x in _scan_inputs(rng, n, 16, 64, 64, 1)]
        q = _t(rng.normal(size=(1, 2, 8, 64)), torch.float16)
        kv = _t(rng.normal(size=(1, 3000 + n, 4, 64)), torch.float16)
        calls.append((a, q, kv))

    def run(a, q, kv):
        state = a[0].clone()
        return kda_prefill(state, *(x[None] for x in a[1:]), scale=0.2), state, attention_prefill(q, kv, kv)

    want = [run(*c) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [None, None]
    for _ in range(3):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = run(*calls[i])
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert all(torch.equal(s, t) for s, t in zip(x, y))
