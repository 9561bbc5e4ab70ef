"""GPU parity of the prompt KDA kernels (local_kimi_amd/csrc/kda_prefill.hip) with oracle/kda.py.

Tolerances, all against float64 on the same inputs:

* convolutions: half a step of the storage dtype (eps / 2 of the value; 2^-25
  for fp16 subnormals) and the fp32 error before it. The sum of four products is
  off by at most 4 * 2^-24 * sum |w x| and silu's slope is below 1.1; its
  exponential takes a rounded argument (|y| 2^-24 relative) and the
  hardware exp2, reciprocal and two products add at most 6 * 2^-24. States
  are copies: exact.
* recurrence: every element of the state gets about six roundings a step
  (2^-24 each at most, a third of that rms), and neither decay <= 0 nor the
  correction (1 - beta k k^T, |k| = 1, 0 <= beta <= 1) enlarges what is there, so after
  L steps the rounding error is at most of rms 2 * 2^-24 * sqrt(L + 16) relative to the
  state's own; twice that is asked for in the 2-norm, and no element beyond eight
  times it. The same holds for the fp32 outputs; 16-bit outputs add
  half a step of their dtype.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kda as K

pytestmark = pytest.mark.gpu

DEV = "cuda"
_NAMES = {torch.float32: "float32", torch.float16: "float16", torch.bfloat16: "bfloat16"}


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from local_kimi_amd import _lib

    _lib.load()


def _t(a, dtype=torch.float32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV, dtype)


def _np(t):
    return t.detach().double().cpu().numpy()


def _cu(lengths):
    return np.concatenate(([0], np.cumsum(lengths))).astype(np.int32)


# ---------------------------------------------------------------------------
# short convolutions


def _conv_inputs(rng, rows, n, c, dtype, wdtype=None):
    def made(shape, std, dt):
        return K.round_to(std * rng.normal(size=shape), _NAMES[dt])

    wdtype = wdtype or dtype
    return ([made((rows, c), 1.0, dtype) for _ in range(3)],
            [made((n, c, 4), 1.0, dtype) for _ in range(3)],
            [made((c, 1, 4), 0.5, wdtype) for _ in range(3)])


def _conv_check(got, x, st, w, dtype, cu, what):
    """got [T, C] against the exact convolution within the derived bound."""
    exact, _ = K.short_conv_prefill(x, st, w, "float32", cu)
    wa = np.abs(w[:, 0])
    size = np.zeros_like(x)  # sum |w x| of each output
    y = np.zeros_like(x)
    for s, (a, b) in enumerate(K.sequence_bounds(cu, x.shape[0], st.shape[0])):
        line = np.concatenate((st[s].T, x[a:b]))
        for j in range(4):
            size[a:b] += np.abs(line[j + 1:j + 1 + b - a]) * wa[:, j]
            y[a:b] += line[j + 1:j + 1 + b - a] * w[:, 0, j]
    fp32 = 2.0 ** -24 * (1.1 * 4 * size + (np.abs(y) + 6 + 1) * np.abs(exact))
    bound = torch.finfo(dtype).eps / 2 * (np.abs(exact) + fp32) + fp32 + 2.0 ** -25 * (
        dtype == torch.float16) + 1e-37
    err = np.abs(_np(got) - exact)
    assert np.all(err <= bound), f"{what}: {(err / bound).max():.3f} of the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lengths,c", [([1], 8), ([3], 2048 + 8), ([33], 72), ([5, 0, 1, 2, 3, 4], 64),
                                       ([64, 31, 32, 33, 1], 16), ([40, 7], 13), ([2, 130], 1)])
def test_conv_matches_oracle(rng, dtype, lengths, c):
    from local_kimi_amd.kernels import short_conv_prefill_triple

    cu, n, rows = _cu(lengths), len(lengths), sum(lengths) + 5  # five rows behind the last
    x, st, w = _conv_inputs(rng, rows, n, c, dtype)
    states = [_t(s, dtype) for s in st]
    outs = short_conv_prefill_triple(*(_t(a[None], dtype) for a in x), *states,
                                     *(_t(a, dtype) for a in w), cu_seqlens=_t(cu, torch.int32))
    for i in range(3):
        _, new = K.short_conv_prefill(x[i], st[i], w[i], "float32", cu)
        assert outs[i].dtype == dtype and outs[i].shape == (1, rows, c)
        _conv_check(outs[i][0], x[i], st[i], w[i], dtype, cu, f"{lengths} {c} {i}")
        assert np.array_equal(_np(states[i]), new)
        assert not outs[i][0, sum(lengths):].any()


def test_conv_state_out_leaves_the_states(rng):
    from local_kimi_amd.kernels import short_conv_prefill_triple

    x, st, w = _conv_inputs(rng, 12, 3, 24, torch.bfloat16)
    args = [[_t(a, torch.bfloat16) for a in part] for part in ([a.reshape(3, 4, 24) for a in x], st, w)]
    kept = [s.clone() for s in args[1]]
    new = [torch.full_like(s, float("nan")) for s in kept]
    a = short_conv_prefill_triple(*args[0], *args[1], *args[2], conv_states_out=tuple(new))
    assert all(torch.equal(s, o) for s, o in zip(args[1], kept))
    b = short_conv_prefill_triple(*args[0], *args[1], *args[2])
    assert all(torch.equal(s, o) for s, o in zip(a, b))
    assert all(torch.equal(s, o) for s, o in zip(args[1], new))


@pytest.mark.parametrize("wdtype", [torch.float32, torch.float16])
def test_conv_takes_views_of_one_projection_and_other_weight_dtypes(rng, wdtype):
    from local_kimi_amd.kernels import short_conv_prefill_triple

    c, n, s = 40, 2, 37
    x, st, w = _conv_inputs(rng, n * s, n, c, torch.bfloat16, wdtype)
    fused = _t(np.concatenate(x, axis=1).reshape(n, s, 3 * c), torch.bfloat16)
    views = fused.split(c, dim=-1)
    assert not views[0].is_contiguous()
    wide = [torch.zeros((n, c, 8), dtype=torch.bfloat16, device=DEV) for _ in range(3)]
    states = [t[..., ::2] for t in wide]  # strided states: updated in place all the same
    for t, a in zip(states, st):
        t.copy_(_t(a, torch.bfloat16))
    outs = short_conv_prefill_triple(*views, *states, *(_t(a[:, 0], wdtype) for a in w))
    for i in range(3):
        _, new = K.short_conv_prefill(x[i], st[i], w[i], "float32")
        _conv_check(outs[i].reshape(n * s, c), x[i], st[i], w[i], torch.bfloat16, None, f"view {i}")
        assert np.array_equal(_np(states[i]), new) and not wide[i][..., 1::2].any()


def test_conv_keeps_infinities_in_their_own_sequence(rng):
    from local_kimi_amd.kernels import short_conv_prefill_triple

    x, st, w = _conv_inputs(rng, 80, 3, 16, torch.bfloat16)
    cu = _t(_cu([30, 20, 30]), torch.int32)

    def run(values):
        states = [_t(a, torch.bfloat16) for a in st]
        outs = short_conv_prefill_triple(*(_t(a[None], torch.bfloat16) for a in values), *states,
                                         *(_t(a, torch.bfloat16) for a in w), cu_seqlens=cu)
        return outs, states

    clean, clean_states = run(x)
    bad = [a.copy() for a in x]
    for a in bad:
        a[30:50] = np.nan
        a[50 - 1] = np.inf
    dirty, dirty_states = run(bad)
    for a, b, sa, sb in zip(clean, dirty, clean_states, dirty_states):
        assert torch.equal(a[0, :30], b[0, :30]) and torch.equal(a[0, 50:], b[0, 50:])
        assert torch.equal(sa[0], sb[0]) and torch.equal(sa[2], sb[2])


# ---------------------------------------------------------------------------
# recurrence


@pytest.fixture(params=["steps", "chunks"])
def form(request):
    """Both forms of the recurrence (d_k above 128 takes steps either way)."""
    from local_kimi_amd import _lib

    with _lib.forced_path("kda_prefill", request.param):
        yield request.param


def _scan_inputs(rng, rows, h, dk, dv, n, dtype=torch.float32, rate=0.1):
    def unit(shape):
        a = rng.normal(size=shape)
        return a / np.linalg.norm(a, axis=-1, keepdims=True)

    a = [0.3 * rng.normal(size=(n, h, dk, dv)), unit((rows, h, dk)), unit((rows, h, dk)),
         K.round_to(rng.normal(size=(rows, h, dv)), _NAMES[dtype]),
         -rate * rng.exponential(size=(rows, h, dk)), 1.0 / (1.0 + np.exp(-rng.normal(size=(rows, h))))]
    return [x.astype(np.float32) for x in a]


def _scan_tol(steps):
    return 4 * 2.0 ** -24 * np.sqrt(steps + 16)


def _close(got, want, steps, dtype, what):
    g = _np(got)
    assert g.shape == want.shape and np.isfinite(g).all(), what
    tol, half = _scan_tol(steps), torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    err = np.abs(g - want)
    rms = np.sqrt(np.mean(want ** 2)) if want.size else 0.0
    step = half * np.abs(want) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    over = np.maximum(err - step, 0.0)
    assert np.sqrt(np.mean(over ** 2)) <= tol * rms + 1e-37, (
        f"{what}: {np.sqrt(np.mean(over ** 2)) / rms:.3g} of the rms, {tol:.3g} allowed")
    assert np.all(over <= 8 * tol * np.maximum(np.abs(want), rms)), f"{what}: {over.max():.3g}"


def _run_scan(a, cu, dtype, scale, **kw):
    from local_kimi_amd.kernels import kda_prefill

    state, q, k, v, decay, beta = a
    st = _t(state)
    out = kda_prefill(st, _t(q[None]), _t(k[None]), _t(v[None], dtype), _t(decay[None]),
                      _t(beta[None]), scale=scale, cu_seqlens=_t(cu, torch.int32), **kw)
    return out[0], st


@pytest.mark.parametrize("lengths,h,dk,dv", [
    ([1], 2, 128, 128), ([2, 0, 17], 3, 64, 64), ([63, 64, 65], 2, 128, 128), ([130], 1, 128, 96),
    ([16, 15, 1, 0, 33], 2, 32, 40), ([70], 2, 72, 30), ([40], 1, 5, 3), ([21, 50], 1, 200, 24),
    ([90], 1, 100, 1), ([300], 2, 128, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_matches_oracle(rng, form, lengths, h, dk, dv, dtype):
    cu, n, rows = _cu(lengths), len(lengths), sum(lengths) + 3
    a = _scan_inputs(rng, rows, h, dk, dv, n, dtype)
    want_state, want = K.prefill(*a, dk ** -0.5, cu)
    out, st = _run_scan(a, cu, dtype, dk ** -0.5)
    assert out.dtype == dtype
    _close(out, want, max(lengths), dtype, f"out {lengths} {h} {dk} {dv}")
    _close(st, want_state, max(lengths), torch.float32, f"state {lengths} {h} {dk} {dv}")
    assert not out[sum(lengths):].any()
    again, st2 = _run_scan(a, cu, dtype, dk ** -0.5)
    assert torch.equal(again, out) and torch.equal(st2, st)


@pytest.mark.parametrize("rate", [0.0, 1e-4, 3.0, 40.0, 1e4])
def test_scan_decays_from_none_to_at_once(rng, form, rate):
    """No decay at all, the usual ones, and ones whose running sums pass what
    an exponential can hold within a few tokens; some channels keep while others fade."""
    cu = _cu([150, 40])
    a = _scan_inputs(rng, 190, 2, 128, 64, 2, rate=rate)
    a[4][:, :, ::3] *= 1e-3
    want_state, want = K.prefill(*a, 0.1, cu)
    out, st = _run_scan(a, cu, torch.float32, 0.1)
    _close(out, want, 150, torch.float32, f"out {rate}")
    _close(st, want_state, 150, torch.float32, f"state {rate}")


def test_scan_infinite_decay_clears_a_channel(rng, form):
    """decay = -inf: the channel's row is forgotten (e^-inf = 0)."""
    cu = _cu([100])
    a = _scan_inputs(rng, 100, 1, 64, 32, 1)
    a[4][::17, :, ::5] = -np.inf
    with np.errstate(invalid="ignore"):
        want_state, want = K.prefill(*a, 1.0, cu)
    out, st = _run_scan(a, cu, torch.float32, 1.0)
    _close(out, want, 100, torch.float32, "out")
    _close(st, want_state, 100, torch.float32, "state")


@pytest.mark.parametrize("beta", [0.0, 1.0])
def test_scan_equal_keys_and_beta_at_its_ends(rng, form, beta):
    """One key for every token: beta = 1 replaces what it holds each step, beta
    = 0 never writes."""
    cu = _cu([140])
    a = _scan_inputs(rng, 140, 1, 128, 32, 1, rate=1e-3)
    a[2][:] = a[2][:1]
    a[5][:] = beta
    want_state, want = K.prefill(*a, 1.0, cu)
    out, st = _run_scan(a, cu, torch.float32, 1.0)
    _close(out, want, 140, torch.float32, "out")
    _close(st, want_state, 140, torch.float32, "state")


def test_scan_keeps_nan_in_its_own_sequence(rng, form):
    cu = _cu([70, 20, 75])
    a = _scan_inputs(rng, 165, 2, 128, 64, 3)
    clean, st = _run_scan(a, cu, torch.float32, 1.0)
    bad = [x.copy() for x in a]
    for x in bad[1:]:
        x[70:90] = np.nan
    dirty, st2 = _run_scan(bad, cu, torch.float32, 1.0)
    assert torch.equal(clean[:70], dirty[:70]) and torch.equal(clean[90:], dirty[90:])
    assert torch.equal(st[0], st2[0]) and torch.equal(st[2], st2[2])
    assert torch.isnan(dirty[70:90]).any()


def test_scan_is_causal_and_splits_into_pieces(rng, form):
    """A prompt in two pieces, the second from the first's state, and a later
    token's change leaving earlier outputs as they were."""
    from local_kimi_amd.kernels import kda_prefill

    a = _scan_inputs(rng, 200, 2, 128, 128, 1)
    want_state, want = K.prefill(*a, 1.0, _cu([200]))
    state, q, k, v, decay, beta = (_t(x if i == 0 else x[None]) for i, x in enumerate(a))
    st = state.clone()
    first = kda_prefill(st, *(t[:, :77] for t in (q, k, v, decay, beta)), scale=1.0)
    second = kda_prefill(st, *(t[:, 77:] for t in (q, k, v, decay, beta)), scale=1.0)
    _close(torch.cat((first, second), 1)[0], want, 200, torch.float32, "pieces")
    _close(st, want_state, 200, torch.float32, "state of the pieces")
    whole = kda_prefill(state.clone(), q, k, v, decay, beta, scale=1.0)
    v2 = v.clone()
    v2[:, 150:] = float("nan")
    later = kda_prefill(state.clone(), q, k, v2, decay, beta, scale=1.0)
    assert torch.equal(whole[:, :150], later[:, :150])


def test_scan_state_out_strided_state_and_batches(rng, form):
    from local_kimi_amd.kernels import kda_prefill

    b, s, h, d = 3, 40, 2, 64
    a = _scan_inputs(rng, b * s, h, d, d, b)
    want_state, want = K.prefill(*a, 0.125)
    args = [_t(x.reshape(b, s, *x.shape[1:])) for x in a[1:]]
    state = _t(a[0])
    new = torch.full_like(state, float("nan"))
    out = kda_prefill(state, *args, scale=0.125, state_out=new)
    _close(out.reshape(b * s, h, d), want, s, torch.float32, "batch")
    _close(new, want_state, s, torch.float32, "state_out")
    assert torch.equal(state, _t(a[0]))
    wide = torch.zeros((b, h, d, 2 * d), device=DEV)
    view = wide[..., ::2]
    view.copy_(state)
    again = kda_prefill(view, *args, scale=0.125)
    assert torch.equal(again, out) and torch.equal(view, new) and not wide[..., 1::2].any()


def test_scan_offsets_outside_the_rows_are_clamped(rng, form):
    """Offsets beyond the rows, decreasing ones and int64 ones."""
    from local_kimi_amd.kernels import kda_prefill

    a = _scan_inputs(rng, 50, 1, 32, 16, 3)
    cu = np.array([0, 30, 20, 900])
    want_state, want = K.prefill(*a, 1.0, cu)
    st = _t(a[0])
    out = kda_prefill(st, *(_t(x[None]) for x in a[1:]), scale=1.0,
                      cu_seqlens=torch.from_numpy(cu).to(DEV))
    # rows 20 to 29 belong to two sequences, whose order is not defined
    _close(out[0, :20], want[:20], 50, torch.float32, "first")
    _close(out[0, 30:], want[30:], 50, torch.float32, "last")
    _close(st, want_state, 50, torch.float32, "states")


# ---------------------------------------------------------------------------
# together


def _layer_inputs(rng, b, s, h, d):
    c = h * d

    def made(shape, std=1.0):
        return _t(std * rng.normal(size=shape), torch.bfloat16)

    return {"in": [made((b, s, c)) for _ in range(3)], "w": [made((c, 1, 4), 0.5) for _ in range(3)],
            "raw_decay": made((b, s, h, d)), "dt_bias": _t(rng.normal(size=h * d) - 3),
            "a_log": _t(np.log(rng.uniform(1, 16, size=(1, 1, h, 1)))), "raw_beta": made((b, s, h))}


def _prompt(d, conv, state, piece, h, dim, cu=None):
    from local_kimi_amd.kernels import (fused_kda_gates, kda_prefill, short_conv_prefill_triple)

    b = d["in"][0].shape[0]
    q, k, v = short_conv_prefill_triple(*(t[:, piece] for t in d["in"]), *conv, *d["w"], cu_seqlens=cu)
    rows = q.shape[1]
    decay, beta, qn, kn = fused_kda_gates(d["raw_decay"][:, piece].contiguous(), d["dt_bias"],
                                          d["a_log"], d["raw_beta"][:, piece].contiguous(), q, k,
                                          num_heads=h, head_dim=dim, eps=1e-6)
    return kda_prefill(state, qn, kn, v.view(b, rows, h, dim), decay, beta, scale=dim ** -0.5,
                       cu_seqlens=cu)


def test_a_prompt_then_decode_tokens_equals_decoding_all_along(rng, form):
    """Convolutions, gates and recurrence over a prompt, then single tokens
    from the states they leave, against the one-launch decode layer token by
    token. bf16 convolution outputs may round apart (an ulp, near ties), which moves
    an output by about eps / 2 of a value now and then."""
    from local_kimi_amd.kernels import kda_decode_layer

    b, s, h, dim = 2, 90, 4, 64
    d = _layer_inputs(rng, b, s + 3, h, dim)

    def fresh():
        conv = [torch.zeros((b, h * dim, 4), dtype=torch.bfloat16, device=DEV) for _ in range(3)]
        return conv, torch.zeros((b, h, dim, dim), device=DEV)

    def token(t, conv, state):
        return kda_decode_layer(*(x[:, t:t + 1].contiguous() for x in d["in"]), *conv, *d["w"],
                                d["raw_decay"][:, t:t + 1].contiguous(), d["dt_bias"], d["a_log"],
                                d["raw_beta"][:, t:t + 1].contiguous(), state, num_heads=h,
                                head_dim=dim)

    conv, state = fresh()
    want = torch.stack([token(t, conv, state) for t in range(s + 3)], 1)
    conv2, state2 = fresh()
    got = [_prompt(d, conv2, state2, slice(0, s), h, dim).float()]
    got += [token(t, conv2, state2)[:, None] for t in range(s, s + 3)]
    got = torch.cat(got, 1)
    for x, y in zip(conv, conv2):
        assert torch.equal(x, y)
    for x, y in ((got, want), (state2, state)):
        assert torch.linalg.norm(x - y) <= 2.0 ** -8 * torch.linalg.norm(y)


def test_graph_replays_match_eager(rng, form):
    """The prompt chain captured once, on padded rows with the offsets in a
    static buffer, replayed for other offsets."""
    h, dim, rows = 4, 64, 150
    d = _layer_inputs(rng, 1, rows, h, dim)
    cu = torch.zeros(4, dtype=torch.int32, device=DEV)
    conv0 = [_t(rng.normal(size=(3, h * dim, 4)), torch.bfloat16) for _ in range(3)]
    state0 = _t(0.1 * rng.normal(size=(3, h, dim, dim)))
    conv, state = [t.clone() for t in conv0], state0.clone()

    def run():
        for t, src in zip(conv, conv0):
            t.copy_(src)
        state.copy_(state0)
        return _prompt(d, conv, state, slice(0, rows), h, dim, cu)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for lengths in ([50, 0, 100], [1, 64, 65], [128, 2, 3], [0, 0, 0]):
        cu.copy_(_t(_cu(lengths), torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got, got_state = out.clone(), state.clone()
        _ = (got_state.float() * 2).sum().item()  # unrelated eager work between replays
        want = run()
        assert torch.equal(got, want) and torch.equal(got_state, state), lengths


def test_calls_on_another_stream(rng, form):
    a = _scan_inputs(rng, 120, 2, 128, 128, 1)
    cu = _cu([120])
    want, want_state = _run_scan(a, cu, torch.float32, 1.0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(_run_scan(a, cu, torch.float32, 1.0))
    torch.cuda.synchronize()
    for out, st in got:
        assert torch.equal(out, want) and torch.equal(st, want_state)
