"""What the prompt operators promise beyond their sums: a query's result does not
depend on what it does not see, finite inputs whose result the type holds give finite
results, states that are only read may be shared, and calls that mix one prompt with
many short sequences.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kda as K

from .test_gpu_attention import _check, _inputs
from .test_gpu_kda_prefill import (DEV, _close, _conv_check, _conv_inputs, _cu, _np, _require_gpu,
                                   _run_scan, _scan_inputs, _t, form)

pytestmark = pytest.mark.gpu

_ = _require_gpu, form  # fixtures


# ---------------------------------------------------------------------------
# attention


@pytest.mark.parametrize("h,hk,d,lk", [(2, 2, 128, 150), (4, 1, 64, 150), (2, 1, 192, 1500)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_later_finite_keys_change_nothing(h, hk, d, lk, dtype):
    """A key of ordinary values that only the later queries of a wave see, large
    enough to be their maximum by far: the earlier queries' results stay as they
    are, bit for bit (their sums have the same terms in the same order), over many
    draws."""
    from local_kimi_amd.kernels import attention_prefill

    lq = 150
    for seed in range(20):
        a = [_t(x[None], dtype) for x in _inputs(np.random.default_rng(seed), lq, lk, h, hk, d, 64, dtype)]
        clean = attention_prefill(*a, scale=0.2)
        for back in (1, 17, 70, 118):  # seen by the last `back` queries
            k = a[1].clone()
            k[:, lk - back] = 8 * a[0][:, lq - 1, ::h // hk, :]
            got = attention_prefill(a[0], k, a[2], scale=0.2)
            assert not torch.equal(got[:, lq - back:], clean[:, lq - back:])
            assert torch.equal(got[:, :lq - back], clean[:, :lq - back]), (seed, back)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_another_heads_queries_change_nothing(dtype):
    """Heads of one key head share a block's rows: a head's result does not
    depend on the other heads' queries."""
    from local_kimi_amd.kernels import attention_prefill

    for seed in range(20):
        a = [_t(x[None], dtype) for x in _inputs(np.random.default_rng(seed), 20, 400, 8, 2, 64, 64, dtype)]
        clean = attention_prefill(*a, scale=0.2)
        q = a[0].clone()
        q[:, :, 1::4] *= 8
        got = attention_prefill(q, *a[1:], scale=0.2)
        for head in (0, 2, 3, 4, 6, 7):
            assert torch.equal(got[:, :, head], clean[:, :, head]), (seed, head)


@pytest.mark.parametrize("keys", [41, 2001])
def test_largest_fp16_values_under_weights_that_round_up(keys):
    """One key of weight 1 and the others just above 1/2, which fp16 rounds up by
    0.9 * 2^-12 each: of forty, 40 * 0.9 * 2^-12 / 21 = 1.7 steps of 2^-12 in their mean,
    where 65504 has one to the next exponent (65520 rounds to infinity). The mean of
    equal values at the type's end is that value; an infinity among them stays one."""
    from local_kimi_amd.kernels import attention_prefill

    q = torch.zeros((1, 41, 1, 64), device=DEV, dtype=torch.float16)
    q[..., 0] = 1
    k = torch.zeros((1, keys, 1, 64), device=DEV, dtype=torch.float16)
    k[:, 1:, :, 0] = -1
    v = torch.full_like(k, 65504.0)
    v[..., 1::2] = -65504.0
    scale = -float(np.log(0.5 + 1.1 * 2.0 ** -12))
    assert torch.equal(attention_prefill(q, k, v, scale=scale), v[:, :41])
    v[:, 0, :, 3] = float("inf")
    got = attention_prefill(q, k, v, scale=scale)
    assert bool((got[..., 3] == float("inf")).all()) and torch.equal(got[..., 4:], v[:, :41, :, 4:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_weights_far_below_the_largest(rng, dtype):
    """4000 keys whose p is 2^-21 or so of the largest one's, below fp16's normal
    range as it is stored: they count, in the sum of the weights as in that of
    the values."""
    from local_kimi_amd.kernels import attention_prefill

    a = _inputs(rng, 1, 4001, 1, 1, 64, 64, dtype)
    a[0][:] = 0.0
    a[0][..., 0] = 1.0
    a[1][:] = 0.0
    a[1][1:, :, 0] = -8.0
    a[2] = np.abs(a[2])
    a[2][0] = 0.0
    scale = 20.6 * float(np.log(2.0)) / 8.0
    got = attention_prefill(*(_t(x[None], dtype) for x in a), scale=scale)
    _check(got, a, scale, dtype, what="far below")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("keys", [150, 2500])
def test_scores_of_minus_infinity(rng, dtype, keys):
    """Keys whose score is -infinity have no weight, and a query that sees no other
    gets zeros; every query here has the sign that makes it so."""
    from local_kimi_amd.kernels import attention_prefill

    a = _inputs(rng, 40, keys, 2, 1, 64, 64, dtype)
    a[0][:, :, 0] = 1.0
    masked = [x.copy() for x in a]
    masked[1][::3, :, 0] = -np.inf
    a[1], a[2] = (np.delete(x, np.arange(0, keys, 3), axis=0) for x in a[1:])
    t = [_t(x[None], dtype) for x in masked]
    got = attention_prefill(t[0][:, -1:], *t[1:])  # (a query that sees every key)
    _check(got, [a[0][-1:], *a[1:]], 0.125, dtype, what="some")
    t[1][..., 0] = -float("inf")
    assert not attention_prefill(*t).any()


@pytest.mark.parametrize("cu_k", [False, True])
def test_attention_of_one_prompt_among_short_ones(rng, cu_k):
    from local_kimi_amd.kernels import attention_prefill

    lengths = [1] * 9 + [700] + [1, 0, 2] * 5
    keys = [n + (5 if n == 1 else 900 if n == 700 else 0) for n in lengths] if cu_k else lengths
    dtype = torch.bfloat16
    a = _inputs(rng, sum(lengths), sum(keys), 4, 2, 64, 64, dtype)
    offsets = {"cu_seqlens": _t(_cu(lengths), torch.int32)}
    if cu_k:
        offsets["cu_seqlens_k"] = _t(_cu(keys), torch.int32)
    got = attention_prefill(*(_t(x[None], dtype) for x in a), **offsets)
    _check(got, a, 0.125, dtype, len(lengths), _cu(lengths), _cu(keys), "mixed")


# ---------------------------------------------------------------------------
# recurrence


@pytest.mark.parametrize("size", [1e-30, 1e30, 1e34, 1e36])
def test_states_of_any_size_that_fp32_holds(rng, form, size):
    """The sums of a step are of a state's size, so a state up to a hundredth of
    fp32's range goes through."""
    cu = _cu([150, 40])
    a = _scan_inputs(rng, 190, 2, 128, 64, 2)
    a[0] *= np.float32(size)
    a[3] *= np.float32(size)
    want_state, want = K.prefill(*a, 0.1, cu)
    out, st = _run_scan(a, cu, torch.float32, 0.1)
    _close(out, want, 150, torch.float32, f"out {size}")
    _close(st, want_state, 150, torch.float32, f"state {size}")


@pytest.mark.parametrize("which", [1, 2])  # q, k
@pytest.mark.parametrize("size", [1e-25, 1e-12, 30.0])
def test_queries_and_keys_of_other_sizes(rng, form, which, size):
    """(Keys above 1 with beta <= 1 / |k|^2, where a step does not enlarge.)"""
    cu = _cu([100, 40])
    a = _scan_inputs(rng, 140, 2, 64, 48, 2)
    a[which] *= np.float32(size)
    if which == 2 and size > 1:
        a[5] /= np.float32(size * size)
    want_state, want = K.prefill(*a, 0.1, cu)
    out, st = _run_scan(a, cu, torch.float32, 0.1)
    _close(out, want, 100, torch.float32, f"out {size}")
    _close(st, want_state, 100, torch.float32, f"state {size}")


@pytest.mark.parametrize("lengths", [[1] * 8 + [500] + [1] * 8, [47], [48], [48, 48, 47], [96, 0],
                                     [300] + [0] * 20])
@pytest.mark.parametrize("dk", [64, 129])
def test_scan_as_it_chooses_its_form(rng, lengths, dk):
    """The form that a call takes by itself, on both sides of its rules."""
    from local_kimi_amd import _lib

    assert _lib.get_path("kda_prefill") == "auto"
    a = _scan_inputs(rng, sum(lengths), 2, dk, 40, len(lengths))
    want_state, want = K.prefill(*a, 0.1, _cu(lengths))
    out, st = _run_scan(a, _cu(lengths), torch.float32, 0.1)
    _close(out, want, max(lengths), torch.float32, "out")
    _close(st, want_state, max(lengths), torch.float32, "state")


# ---------------------------------------------------------------------------
# states


def _conv_call(x, states, w, **kw):
    from local_kimi_amd.kernels import short_conv_prefill_triple

    return short_conv_prefill_triple(*x, *states, *w, **kw)


def test_one_fresh_state_for_the_three_convolutions(rng):
    """States that are only read may be one tensor (and one row for all
    sequences)."""
    n, s, c = 2, 21, 32
    x, st, w = _conv_inputs(rng, n * s, n, c, torch.bfloat16)
    xs = [_t(a.reshape(n, s, c), torch.bfloat16) for a in x]
    ws = [_t(a, torch.bfloat16) for a in w]
    zero = torch.zeros((n, c, 4), device=DEV, dtype=torch.bfloat16)
    for state in (zero, zero[:1].expand(n, c, 4)):
        new = [torch.empty_like(zero) for _ in range(3)]
        outs = _conv_call(xs, [state] * 3, ws, conv_states_out=tuple(new))
        assert not state.any()
        for i in range(3):
            none = np.zeros_like(st[i])
            _conv_check(outs[i].reshape(n * s, c), x[i], none, w[i], torch.bfloat16, None, f"conv {i}")
            assert np.array_equal(_np(new[i]), K.short_conv_prefill(x[i], none, w[i], "float32")[1])


def test_states_that_share_memory_are_refused(rng):
    """A written state that shares a byte with another one, dense or strided."""
    from local_kimi_amd.kernels import kda_prefill

    n, s, c = 2, 5, 32
    x, _, w = _conv_inputs(rng, n * s, n, c, torch.bfloat16)
    xs = [_t(a.reshape(n, s, c), torch.bfloat16) for a in x]
    ws = [_t(a, torch.bfloat16) for a in w]
    wide = torch.zeros((n, 4 * c, 8), device=DEV, dtype=torch.bfloat16)
    one = wide[:, :c, ::2]
    dense = [torch.zeros((n, c, 4), device=DEV, dtype=torch.bfloat16) for _ in range(3)]
    for states, out in (([one] * 3, None), ([dense[0], one, one], None),
                        ([wide[:, i:c + i, ::2] for i in range(3)], None),
                        ([one, *dense[1:]], (one, *dense[1:])), (dense, (one, one, wide[:, c:2 * c, ::2])),
                        (dense, (dense[0], one, wide[:, c:2 * c, ::2])), ([dense[0]] * 3, None)):
        with pytest.raises(ValueError, match="overlap"):
            _conv_call(xs, states, ws, conv_states_out=out)
    state = torch.zeros((n, 2, 16, 16), device=DEV)[..., ::2]
    args = [torch.zeros((n, s, 2, width), device=DEV) for width in (16, 16, 8, 16)]
    with pytest.raises(ValueError, match="overlap"):
        kda_prefill(state, *args, torch.zeros((n, s, 2), device=DEV), scale=1.0, state_out=state)


def test_states_beside_each_other_in_one_buffer(rng):
    """Interleaved and neighbouring views of one buffer share no byte."""
    n, s, c = 3, 9, 24
    x, st, w = _conv_inputs(rng, n * s, n, c, torch.bfloat16)
    xs = [_t(a.reshape(n, s, c), torch.bfloat16) for a in x]
    ws = [_t(a, torch.bfloat16) for a in w]
    for views in (lambda b: [b[:, i * c:(i + 1) * c, :4] for i in range(3)],
                  lambda b: [b[:, i:3 * c:3, :4] for i in range(3)],
                  lambda b: [b[:, :c, ::2], b[:, :c, 1::2], b[:, c:2 * c, ::2]]):
        buffer = torch.zeros((n, 3 * c, 8), device=DEV, dtype=torch.bfloat16)
        states = views(buffer)
        for t, a in zip(states, st):
            t.copy_(_t(a, torch.bfloat16))
        _conv_call(xs, states, ws)
        for i in range(3):
            want = K.short_conv_prefill(x[i], st[i], w[i], "float32")[1]
            assert np.array_equal(_np(states[i]), want)
