"""Refusals of the prompt operators, in Python and at the C ABI: all on the host,
before any launch, so they run without a GPU."""

from __future__ import annotations

import pytest
import torch

from local_kimi_amd import _lib
from local_kimi_amd.kernels import attention_prefill, kda_prefill, short_conv_prefill_triple


def _conv(b=2, s=5, c=16, n=None, dtype=torch.bfloat16):
    n = b if n is None else n
    return ([torch.zeros(b, s, c, dtype=dtype) for _ in range(3)],
            [torch.zeros(n, c, 4, dtype=dtype) for _ in range(3)],
            [torch.zeros(c, 1, 4, dtype=dtype) for _ in range(3)])


def test_conv_refusals():
    x, st, w = _conv()
    call = short_conv_prefill_triple
    with pytest.raises(ValueError, match="CUDA"):
        call(*x, *st, *w)
    with pytest.raises(ValueError, match="shape \\[batch, sequence, channels\\]"):
        call(x[0][0], *x[1:], *st, *w)
    with pytest.raises(ValueError, match="identical shapes"):
        call(x[0][:, :3], *x[1:], *st, *w)
    with pytest.raises(ValueError, match="state must have shape"):
        call(*x, st[0][:1], *st[1:], *w)
    with pytest.raises(ValueError, match="weight must have shape"):
        call(*x, *st, w[0][:3], *w[1:])
    with pytest.raises(TypeError, match="share a dtype"):
        call(*x, st[0].float(), *st[1:], *w)
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        call(*(t.double() for t in x), *(t.double() for t in st), *w)
    with pytest.raises(ValueError, match="nonempty batch"):
        call(*(t[:0] for t in x), *(t[:0] for t in st), *w)


def test_offsets_refusals():
    x, st, w = _conv(1, 9, 16, 3)
    for cu, error in ((torch.zeros(1, dtype=torch.int32), ValueError),
                      (torch.zeros((2, 2), dtype=torch.int32), ValueError),
                      (torch.zeros(4), TypeError)):
        with pytest.raises(error, match="cu_seqlens"):
            short_conv_prefill_triple(*x, *st, *w, cu_seqlens=cu)
    x, st, w = _conv(2, 9, 16, 3)
    with pytest.raises(ValueError, match="batch one"):
        short_conv_prefill_triple(*x, *st, *w, cu_seqlens=torch.zeros(4, dtype=torch.int32))


def test_scan_refusals():
    b, s, h, d = 2, 4, 3, 16
    state = torch.zeros(b, h, d, d)
    q, k, v, g = (torch.zeros(b, s, h, d) for _ in range(4))
    beta = torch.zeros(b, s, h)
    ok = {"scale": 1.0}
    with pytest.raises(ValueError, match="CUDA"):
        kda_prefill(state, q, k, v, g, beta, **ok)
    with pytest.raises(TypeError, match="float32"):
        kda_prefill(state, q.half(), k, v, g, beta, **ok)
    with pytest.raises(TypeError, match="v must be"):
        kda_prefill(state, q, k, v.double(), g, beta, **ok)
    with pytest.raises(ValueError, match="k must have shape"):
        kda_prefill(state, q, k[:, :1], v, g, beta, **ok)
    with pytest.raises(ValueError, match="decay must have shape"):
        kda_prefill(state, q, k, v, g[..., :8], beta, **ok)
    with pytest.raises(ValueError, match="beta must have shape"):
        kda_prefill(state, q, k, v, g, beta[..., :2], **ok)
    with pytest.raises(ValueError, match="v must have shape"):
        kda_prefill(state, q, k, v[:, :2], g, beta, **ok)
    with pytest.raises(ValueError, match="state must have shape"):
        kda_prefill(state[:1], q, k, v, g, beta, **ok)
    with pytest.raises(ValueError, match="overlaps"):
        kda_prefill(state, q, k, v, g, beta, state_out=state, **ok)
    with pytest.raises(ValueError, match="match the state"):
        kda_prefill(state, q, k, v, g, beta, state_out=state.double(), **ok)


def test_attention_refusals():
    def made(b=1, s=6, sk=6, h=4, hk=2, dq=64, dv=64, dtype=torch.bfloat16):
        return (torch.zeros(b, s, h, dq, dtype=dtype), torch.zeros(b, sk, hk, dq, dtype=dtype),
                torch.zeros(b, sk, hk, dv, dtype=dtype))

    with pytest.raises(ValueError, match="CUDA"):
        attention_prefill(*made())
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        attention_prefill(*made(dtype=torch.float32))
    q, k, v = made()
    with pytest.raises(TypeError, match="share one dtype"):
        attention_prefill(q, k.half(), v)
    with pytest.raises(ValueError, match="multiple of the key heads"):
        attention_prefill(*made(h=3))
    for dims in ({"dq": 200}, {"dq": 60}):
        with pytest.raises(ValueError, match="d_qk"):
            attention_prefill(*made(**dims))
    for dims in ({"dv": 136}, {"dv": 12}):
        with pytest.raises(ValueError, match="d_v"):
            attention_prefill(*made(**dims))
    with pytest.raises(ValueError, match="k must have shape"):
        attention_prefill(q, k[:, :3], v)
    with pytest.raises(ValueError, match="shape \\[batch"):
        attention_prefill(q[0], k[0], v[0])
    cu = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="needs cu_seqlens"):
        attention_prefill(q, k, v, cu_seqlens_k=cu)
    with pytest.raises(ValueError, match="same length"):
        attention_prefill(q, k, v, cu_seqlens=cu, cu_seqlens_k=cu[:2])
    with pytest.raises(ValueError, match="need cu_seqlens_k"):
        attention_prefill(*made(sk=9), cu_seqlens=cu)
    with pytest.raises(ValueError, match="finite"):
        attention_prefill(q, k, v, scale=float("inf"))


@pytest.fixture(scope="module")
def lib():
    if not _lib.is_built():
        pytest.skip("library not built; run python -m local_kimi_amd._build")
    return _lib.load()


def test_c_abi_refusals_come_before_any_launch(lib):
    """The pointers here are never dereferenced."""
    def conv(seqs=1, tokens=8, c=8, stride=8, vd=2, wd=2, p=16):
        _lib.call("lk_kda_short_conv_prefill", *([p] * 15), None, seqs, tokens, c, stride, vd, wd,
                  None)

    for args, match in (({"seqs": 0}, "sequences"), ({"seqs": 3}, "divide"), ({"c": 0}, "channels"),
                        ({"stride": 7}, "stride"), ({"vd": 3}, "dtype"), ({"wd": -1}, "dtype"),
                        ({"p": None}, "null"), ({"p": 2}, "aligned"), ({"tokens": 1 << 31}, "too many")):
        with pytest.raises(RuntimeError, match=match):
            conv(**args)

    def scan(seqs=1, tokens=8, h=2, dk=64, dv=64, vd=0, p=16):
        _lib.call("lk_kda_prefill", *([p] * 8), None, seqs, tokens, h, dk, dv, 1.0, vd, None, 0, None)

    for args, match in (({"seqs": 3}, "divide"), ({"h": 0}, "nonzero"), ({"dk": 257}, "d_k up to 256"),
                        ({"vd": 7}, "dtype"), ({"p": None}, "null"), ({"p": 8}, "16-byte")):
        with pytest.raises(RuntimeError, match=match):
            scan(**args)

    def attention(seqs=1, tq=8, tk=8, h=4, hk=2, dq=64, dv=64, stride=256, scale=1.0, dt=2, p=16):
        _lib.call("lk_attention_prefill", p, p, p, p, None, None, seqs, tq, tk, h, hk, dq, dv,
                  stride, dq, stride, dq, stride, dv, scale, dt, None, 0, None)

    for args, match in (({"seqs": 3}, "divide"), ({"hk": 3}, "multiple of the key heads"),
                        ({"dq": 200}, "d_qk"), ({"dv": 136}, "d_v"), ({"dt": 0}, "fp16 or bf16"),
                        ({"stride": 12}, "multiples of 8"), ({"stride": -8}, "negative"),
                        ({"scale": float("nan")}, "finite"), ({"p": None}, "null"),
                        ({"p": 8}, "16-byte")):
        with pytest.raises(RuntimeError, match=match):
            attention(**args)
    assert lib.lk_kda_prefill_workspace(0, 8, 2, 64, 64) == -1
    assert lib.lk_attention_prefill_workspace(8, 8, 1, 3, 2, 64, 64) == -1
