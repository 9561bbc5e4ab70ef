"""GPU parity of causal prompt attention (local_kimi_amd/csrc/attention.hip) with oracle/attention.py.

Tolerance, element by element against float64 on the same inputs: p is rounded
to the inputs' dtype for its product (at most eps / 2 of each term, so eps / 2 *
sum p |v|) and the output once more (eps / 2 of it). Before that all is
fp32: a score is off by at most (d_qk + 4) * 2^-24 of scale * sum |q| |k|, twice that
in p (the score and the maximum it is taken against), and the sums of p and
p v by at most 2^-24 a key seen.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.attention import attention_prefill as oracle_attention
from oracle.kda import round_to

pytestmark = pytest.mark.gpu

DEV = "cuda"
_NAMES = {torch.float16: "float16", torch.bfloat16: "bfloat16"}


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from local_kimi_amd import _lib

    _lib.load()


def _t(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV, dtype)


def _cu(lengths):
    return np.concatenate(([0], np.cumsum(lengths))).astype(np.int32)


def _inputs(rng, tq, tk, h, hk, dq, dv, dtype, std=1.0):
    return [round_to(std * rng.normal(size=s), _NAMES[dtype])
            for s in ((tq, h, dq), (tk, hk, dq), (tk, hk, dv))]


def _bound(out, spread, score, keys, d_qk, dtype):
    half = torch.finfo(dtype).eps / 2
    fp32 = 2.0 ** -24 * (2 * (d_qk + 4) * score[..., None] + keys + 8) * spread
    return half * (1 + half) * (spread + np.abs(out)) + 1.1 * fp32 + 2.0 ** -25


def _check(got, arrays, scale, dtype, sequences=1, cu_q=None, cu_k=None, what=""):
    out, spread, score = oracle_attention(*arrays, scale, sequences, cu_q, cu_k)
    g = got.detach().double().cpu().numpy().reshape(out.shape)
    assert got.dtype == dtype
    bound = _bound(out, spread, score, arrays[1].shape[0], arrays[0].shape[-1], dtype)
    err = np.abs(g - out)
    assert np.isfinite(g).all() and np.all(err <= bound), (
        f"{what}: {np.nanmax(err / bound):.3f} of the bound")


@pytest.mark.parametrize("h,hk,dq,dv", [(2, 2, 192, 128), (4, 1, 128, 128), (6, 3, 64, 64),
                                        (2, 1, 72, 40), (1, 1, 8, 8), (2, 2, 136, 64), (2, 2, 64, 128)])
@pytest.mark.parametrize("lengths", [[1], [2, 0, 63], [64], [65, 1, 127], [130, 129]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed_prompts_match_oracle(rng, h, hk, dq, dv, lengths, dtype):
    from local_kimi_amd.kernels import attention_prefill

    rows = sum(lengths) + 3
    a = _inputs(rng, rows, rows, h, hk, dq, dv, dtype)
    cu = _cu(lengths)
    got = attention_prefill(*(_t(x[None], dtype) for x in a), cu_seqlens=_t(cu, torch.int32))
    _check(got, a, dq ** -0.5, dtype, len(lengths), cu, cu, f"{lengths} {h}/{hk} {dq}/{dv}")
    assert not got[0, sum(lengths):].any()
    again = attention_prefill(*(_t(x[None], dtype) for x in a), cu_seqlens=_t(cu, torch.int32))
    assert torch.equal(got, again)


@pytest.mark.parametrize("lq,lk", [([1, 5, 40], [300, 700, 41]), ([33], [1500]), ([20, 7], [5, 0]),
                                   ([1], [1]), ([150], [333]), ([0, 4], [9, 4]), ([1] * 5, [1000, 1, 64, 65, 0])])
@pytest.mark.parametrize("h,hk,dq,dv", [(2, 2, 192, 128), (4, 2, 64, 64)])
def test_keys_before_the_queries(rng, lq, lk, h, hk, dq, dv):
    """Continued prompts; where there are fewer keys than queries the first see none."""
    from local_kimi_amd.kernels import attention_prefill

    dtype = torch.bfloat16
    a = _inputs(rng, sum(lq) + 2, sum(lk) + 1, h, hk, dq, dv, dtype)
    cu, cuk = _cu(lq), _cu(lk)
    got = attention_prefill(*(_t(x[None], dtype) for x in a), cu_seqlens=_t(cu, torch.int64),
                            cu_seqlens_k=_t(cuk, torch.int32), scale=0.2)
    _check(got, a, 0.2, dtype, len(lq), cu, cuk, f"{lq} {lk}")
    assert not got[0, sum(lq):].any()


@pytest.mark.parametrize("b,s,sk", [(3, 50, 50), (2, 10, 200), (2, 6, 3), (2, 1, 130)])
def test_batches_of_equal_sequences(rng, b, s, sk):
    from local_kimi_amd.kernels import attention_prefill

    dtype = torch.float16
    a = _inputs(rng, b * s, b * sk, 4, 2, 64, 64, dtype)
    got = attention_prefill(*(_t(x.reshape(b, -1, *x.shape[1:]), dtype) for x in a))
    _check(got, a, 64 ** -0.5, dtype, b, None, None, f"{b} {s} {sk}")


@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0])
def test_sharp_negative_and_flat_scores(rng, scale):
    """Scores of some hundreds (one key takes all), a negative scale, none at all."""
    from local_kimi_amd.kernels import attention_prefill

    dtype = torch.bfloat16
    a = _inputs(rng, 200, 200, 1, 1, 128, 128, dtype, std=3.0)
    got = attention_prefill(*(_t(x[None], dtype) for x in a), scale=scale)
    _check(got, a, scale, dtype, what=f"scale {scale}")


def test_scores_that_overflow_an_exponential_without_its_maximum(rng):
    """fp16 values near the top of the type: scores beyond 1e4."""
    from local_kimi_amd.kernels import attention_prefill

    dtype = torch.float16
    a = _inputs(rng, 70, 70, 2, 1, 64, 64, dtype, std=30.0)
    a[2] = round_to(a[2] * 500.0, "float16")
    got = attention_prefill(*(_t(x[None], dtype) for x in a))
    _check(got, a, 64 ** -0.5, dtype, what="large")


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), torch.finfo(torch.bfloat16).min])
def test_what_a_query_does_not_see_has_no_part(rng, bad):
    """Bad values in later keys and values, and in other sequences."""
    from local_kimi_amd.kernels import attention_prefill

    dtype = torch.bfloat16
    lengths = [100, 37, 150]
    a = [_t(x[None], dtype) for x in _inputs(rng, 287, 287, 2, 1, 192, 128, dtype)]
    cu = _t(_cu(lengths), torch.int32)
    clean = attention_prefill(*a, cu_seqlens=cu)
    for spots in (list(range(100, 137)), [70], [99], [286], [137 + 64], [137 + 20, 137 + 21]):
        k, v = a[1].clone(), a[2].clone()
        k[:, spots] = bad
        v[:, spots] = bad
        got = attention_prefill(a[0], k, v, cu_seqlens=cu)
        at = 0
        for n in lengths:
            first = min((s for s in spots if at <= s < at + n), default=at + n)
            assert torch.equal(got[:, at:first], clean[:, at:first]), (spots, at)
            at += n


def test_strided_and_expanded_inputs(rng):
    """Slices of one fused projection, a rotary part shared by the heads, and
    layouts that have to be copied."""
    from local_kimi_amd.kernels import attention_prefill

    dtype = torch.bfloat16
    b, s, h = 2, 70, 4
    fused = torch.randn((b, s, h, 192 + 192 + 128), device=DEV).to(dtype)
    q, k, v = fused.split([192, 192, 128], dim=-1)
    want = attention_prefill(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(attention_prefill(q, k, v), want)
    one = k[:, :, :1].expand(b, s, h, 192)
    assert torch.equal(attention_prefill(q, one, v),
                       attention_prefill(q.contiguous(), one.contiguous(), v.contiguous()))
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(attention_prefill(*heads_first), want)
    odd = torch.zeros((b, s, h, 193), device=DEV, dtype=dtype)[..., 1:]
    odd.copy_(q)
    assert torch.equal(attention_prefill(odd, k, v), want)


def test_graph_replays_with_other_lengths(rng):
    from local_kimi_amd.kernels import attention_prefill

    dtype = torch.bfloat16
    a = [_t(x[None], dtype) for x in _inputs(rng, 300, 300, 2, 1, 128, 128, dtype)]
    cu = torch.zeros(4, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attention_prefill(*a, cu_seqlens=cu)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of one call, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attention_prefill(*a, cu_seqlens=cu))
        graphs.append(g)
    for lengths in ([100, 0, 200], [1, 1, 1], [299, 1, 0], [128, 128, 44], [0, 0, 0]):
        cu.copy_(_t(_cu(lengths), torch.int32))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = attention_prefill(*a, cu_seqlens=cu)
        _ = (want.float() * 2).sum().item()  # unrelated eager work between replays
        for o in outs:
            assert torch.equal(o, want), lengths


def test_long_prompt_against_float64_on_the_gpu(rng):
    """2500 tokens, grouped heads: the loop's many passes and every XCD's share."""
    from local_kimi_amd.kernels import attention_prefill

    dtype, s, h, hk = torch.bfloat16, 2500, 10, 5
    g = torch.Generator(device=DEV).manual_seed(7)
    q, k, v = (torch.randn((1, s, n, d), generator=g, device=DEV).to(dtype)
               for n, d in ((h, 192), (hk, 192), (hk, 128)))
    got = attention_prefill(q, k, v)[0].double()
    mask = torch.ones((s, s), dtype=torch.bool, device=DEV).tril()
    half = torch.finfo(dtype).eps / 2
    for head in range(h):
        qh, kh, vh = (t[0, :, i].double() for t, i in ((q, head), (k, head // 2), (v, head // 2)))
        score = (qh @ kh.t().contiguous()) * 192 ** -0.5
        size = 192 ** -0.5 * (qh.abs() @ kh.abs().t().contiguous()).amax(1, keepdim=True)
        p = torch.softmax(score.masked_fill(~mask, float("-inf")), -1)
        want, spread = p @ vh, p @ vh.abs()
        bound = half * (1 + half) * (spread + want.abs()) \
            + 1.1 * 2.0 ** -24 * (2 * 196 * size + s + 8) * spread + 2.0 ** -25
        err = (got[:, head] - want).abs()
        assert bool((err <= bound).all()), f"head {head}: {(err / bound).max().item():.3f}"
