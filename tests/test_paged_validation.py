"""Refusals of the paged-cache operators, in Python and at the C ABI: all on the host,
before any launch, so they run without a GPU. The oracle's two forms against each other."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from local_kimi_amd import _lib
from local_kimi_amd.kernels import (attention_paged, copy_pages, paged_append, qk_norm_rope,
                                    qk_norm_rope_append, rope_table)
from oracle import paged as P

BF = torch.bfloat16


def _heads(b=1, s=6, h=4, hk=2, d=64, dv=64, dtype=BF):
    return (torch.zeros(b, s, h, d, dtype=dtype), torch.zeros(b, s, hk, d, dtype=dtype),
            torch.zeros(b, s, hk, dv, dtype=dtype))


def _cache(n=1, pages=5, rows=16, hk=2, d=64, dv=64, dtype=BF):
    return (torch.zeros(pages, rows, hk, d, dtype=dtype), torch.zeros(pages, rows, hk, dv, dtype=dtype),
            torch.zeros(n, 3, dtype=torch.int32), torch.zeros(n, dtype=torch.int32))


def test_rope_refusals():
    q, k, _ = _heads()
    cs, at = torch.zeros(9, 64), torch.zeros(1, 6, dtype=torch.int32)
    w = torch.ones(64)
    with pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope(q, k, cs, at)
    for args, error, match in (
            ((q[0], k, cs, at), ValueError, "shape \\[batch"), ((q, k[:, :3], cs, at), ValueError, "agree"),
            ((q, k.half(), cs, at), TypeError, "one dtype"),
            ((q.double(), k.double(), cs, at), TypeError, "float32, float16 or bfloat16"),
            ((q[..., :60], k[..., :60], cs, at), ValueError, "multiple of 8"),
            ((q[:, :, :0], k, cs, at), ValueError, "nonzero"),
            ((q, k, cs.half(), at), TypeError, "cos_sin must be float32"),
            ((q, k, cs[0], at), ValueError, "cos_sin must have shape"),
            ((q, k, cs[:0], at), ValueError, "cos_sin must have shape"),
            ((q, k, cs[:, :12], at), ValueError, "rotated slice"),
            ((q, k, torch.zeros(9, 72), at), ValueError, "rotated slice"),
            ((q, k, cs, at[:, :5]), ValueError, "positions must have shape"),
            ((q, k, cs, at.float()), TypeError, "positions must be"),
            ((q, k, cs, at, w), ValueError, "both be given"),
            ((q, k, cs, at, w, w[:8]), ValueError, "norm weights must have shape"),
            ((q, k, cs, at, w, w.half()), TypeError, "share one dtype"),
            ((q, k, cs, at, w, w, -1.0), ValueError, "eps"),
            ((q, k, cs, at, w, w, float("nan")), ValueError, "eps")):
        with pytest.raises(error, match=match):
            qk_norm_rope(*args)
    for offset in (4, 8, -8):
        with pytest.raises(ValueError, match="rotated slice"):
            qk_norm_rope(q, k, cs, at, rotary_offset=offset)
    with pytest.raises(ValueError, match="multiple of 8"):
        rope_table(9, 12)


def test_append_refusals():
    q, k, v = _heads()
    kp, vp, table, lengths = _cache()
    cs = torch.zeros(9, 64)

    def call(q=q, k=k, v=v, kp=kp, vp=vp, table=table, lengths=lengths, **kw):
        qk_norm_rope_append(q, k, v, kp, vp, table, lengths, cs, **kw)

    cu = torch.zeros(3, dtype=torch.int32)
    for kw, error, match in (
            ({}, ValueError, "CUDA"), ({"v": v[:, :2]}, ValueError, "v must have shape"),
            ({"v": v.half()}, TypeError, "share one dtype"), ({"v": v[..., :32]}, ValueError, "cache's width"),
            ({"kp": kp[0]}, ValueError, "k_pages and v_pages must have shape"),
            ({"vp": vp[:4]}, ValueError, "k_pages and v_pages must have shape"),
            ({"kp": kp[:, :8], "vp": vp[:, :8]}, ValueError, "multiple of 16 rows"),
            ({"kp": kp[:, :0], "vp": vp[:, :0]}, ValueError, "multiple of 16 rows"),
            ({"kp": kp[:, :, :1], "vp": vp[:, :, :1]}, ValueError, "the cache holds"),
            ({"kp": kp[..., :32]}, ValueError, "the cache holds"), ({"kp": kp.half()}, TypeError, "inputs' dtype"),
            ({"table": table[0]}, ValueError, "page_table must have shape"),
            ({"lengths": lengths[None]}, ValueError, "page_table must have shape"),
            ({"table": table.long()}, TypeError, "int32"), ({"lengths": lengths.float()}, TypeError, "int32"),
            ({"kp": torch.zeros(5, 16, 2, 65, dtype=BF)[..., 1:]}, ValueError, "16 bytes"),
            ({"kp": torch.zeros(5, 16, 64, 2, dtype=BF).transpose(2, 3)}, ValueError, "dense"),
            ({"cu_seqlens": cu}, ValueError, "the table has 1 sequences, the call 2"),
            ({"cu_seqlens": cu.float()}, TypeError, "cu_seqlens")):
        with pytest.raises(error, match=match):
            call(**kw)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        paged_append(k.float(), v.float(), kp.float(), vp.float(), table, lengths)
    with pytest.raises(ValueError, match="the table has 1"):
        paged_append(*(t.expand(2, -1, -1, -1) for t in (k, v)), kp, vp, table, lengths)
    with pytest.raises(ValueError, match="CUDA"):
        paged_append(k, v, kp, vp, table, lengths)


def test_attention_refusals():
    q = _heads()[0]
    kp, vp, table, lengths = _cache()
    for args, error, match in (
            ((q, kp, vp, table, lengths), ValueError, "CUDA"),
            ((q.float(), kp, vp, table, lengths), TypeError, "float16 or bfloat16"),
            ((q.half(), kp, vp, table, lengths), TypeError, "inputs' dtype"),
            ((q[0], kp, vp, table, lengths), ValueError, "shape \\[batch"),
            ((q[:, :, :3], kp, vp, table, lengths), ValueError, "multiple of the key heads"),
            ((q, kp[0], vp, table, lengths), ValueError, "multiple of the key heads"),
            ((q[..., :60], kp[..., :60], vp, table, lengths), ValueError, "d_qk"),
            ((torch.zeros(1, 2, 4, 200, dtype=BF), torch.zeros(5, 16, 2, 200, dtype=BF), vp, table, lengths),
             ValueError, "d_qk"),
            ((q, kp, torch.zeros(5, 16, 2, 136, dtype=BF), table, lengths), ValueError, "d_v"),
            ((q, kp, vp, table.expand(2, -1), lengths.expand(2)), ValueError, "the table has 2")):
        with pytest.raises(error, match=match):
            attention_paged(*args)
    with pytest.raises(ValueError, match="finite"):
        attention_paged(q, kp, vp, table, lengths, scale=float("nan"))


def test_copy_refusals():
    t = torch.zeros(6, 16, 2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        copy_pages([t], [0], [1])
    for args, match in ((([t], [0, 1], [2]), "one length"), (([t, t[:4]], [0], [1]), "one number of pages"),
                        (([t[..., :4]], [0], [1]), "dense"), (([t[:, :, 0]], [0], [1]), "dense"),
                        (([torch.zeros(6, 3)], [0], [1]), "16 bytes"),
                        (([torch.zeros(1, 16, 2, 8).expand(6, 16, 2, 8)], [0], [1]), "must not overlap"),
                        (([torch.zeros(6)], [0], [1]), "shape"), (([torch.tensor(0.0)], [0], [1]), "shape"),
                        (([t], [2 ** 31], [1]), "beyond"), (([t], torch.zeros(1), [1]), "integers on the host"),
                        (([t], torch.zeros(1, 1, dtype=torch.int64), [1]), "integers on the host")):
        with pytest.raises(ValueError, match=match):
            copy_pages(*args)
    with pytest.raises(TypeError):
        copy_pages([t], [0.5], [1])


@pytest.fixture(scope="module")
def lib():
    if not _lib.is_built():
        pytest.skip("library not built; run python -m local_kimi_amd._build")
    return _lib.load()


def test_c_abi_refusals_come_before_any_launch(lib):
    """The pointers here are never dereferenced."""
    def rope(rows=8, h=4, hk=2, d=64, stride=256, rotary=64, offset=0, table=9, eps=1e-6, dt=2, wd=0, p=16, w=16):
        _lib.call("lk_qk_norm_rope", p, p, w, w, p, p, p, p, rows, h, hk, d, stride, d, stride, d, rotary,
                  offset, 0, table, 0, eps, dt, wd, None)

    for args, match in (({"rows": -1}, "rows"), ({"rows": 1 << 31}, "rows"), ({"h": 0}, "heads"), ({"hk": 0}, "heads"),
                        ({"h": 65536}, "heads"), ({"d": 264}, "head dimension"), ({"d": 60}, "head dimension"),
                        ({"stride": 12}, "multiples of 8"), ({"stride": -8}, "not negative"),
                        ({"rotary": 72}, "rotated slice"), ({"rotary": 12}, "rotated slice"),
                        ({"offset": 8}, "rotated slice"), ({"offset": -8}, "rotated slice"),
                        ({"table": 0}, "table of angles"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"),
                        ({"dt": 3}, "dtype"), ({"wd": 3}, "dtype"), ({"p": None, "rotary": 0}, "null"),
                        ({"p": 8, "rotary": 0}, "16-byte"), ({"w": 8}, "16-byte"),
                        ({"rows": (1 << 31) - 1, "h": 65535}, "too many rows and heads")):
        with pytest.raises(RuntimeError, match=match):
            rope(**args)

    def append(seqs=1, rows=8, h=4, hk=2, d=64, dv=64, pages=5, page_rows=16, width=3, stride=3, page=4096,
               row=128, rotary=64, dt=2, p=16, q=16, vp=32, head=64):
        _lib.call("lk_paged_append", q, p, p, p, p, 16, p, p, None, q, p, vp if p else p, seqs, rows, h, hk, d, dv, 256, d,
                  128, d, 128, dv, pages, page_rows, width, stride, page, row, head, page, row, head, rotary, 0, 0,
                  9, 1e-6, dt, 0, None)

    shared = (({"seqs": 0}, "sequences"), ({"seqs": 1 << 24, "rows": 0}, "sequences"), ({"seqs": 3}, "divide"),
              ({"pages": -1}, "pages"), ({"pages": 1 << 31}, "pages"), ({"page_rows": 24}, "multiple of 16"),
              ({"page_rows": 0}, "multiple of 16"), ({"page_rows": 65552}, "multiple of 16"),
              ({"width": (1 << 26) + 1, "stride": 1 << 27}, "up to 2\\^30"), ({"stride": 2}, "page table"),
              ({"width": 1 << 62, "stride": 1 << 62}, "up to 2\\^30"), ({"page": 4}, "multiples of 8"),
              ({"row": -8}, "not negative"), ({"p": None}, "null"), ({"p": 8}, "16-byte"), ({"dt": 0}, "fp16"))
    for args, match in (*shared, ({"q": None}, "null"), ({"page": 0}, "overlap"), ({"row": 64}, "overlap"),
                        ({"page": 2000}, "overlap"), ({"head": 56}, "overlap"), ({"vp": 16}, "pages of their own"), ({"dv": 264}, "value dimension"), ({"dv": 12}, "value dimension"),
                        ({"rotary": 72}, "rotated slice")):
        with pytest.raises(RuntimeError, match=match):
            append(**args)
    append(rows=0)
    append(rows=0, head=16 * 64, row=64, page=32 * 64)  # heads first
    append(rows=0, page=128, row=5 * 128)                # rows of all pages side by side

    def attention(seqs=1, rows=8, h=4, hk=2, d=64, dv=64, pages=5, page_rows=16, width=3, stride=3, page=4096,
                  row=128, scale=1.0, dt=2, p=16, qs=256, ws=None, size=0):
        _lib.call("lk_attention_paged", p, p, p, p, p, p, None, seqs, rows, h, hk, d, dv, qs, d, pages, page_rows,
                  width, stride, page, row, d, page, row, dv, scale, dt, ws, size, None)

    long = {"width": 100, "stride": 100}
    need = lib.lk_attention_paged_workspace(8, 1, 1600, 4, 2, 64, 64, 0)
    assert need > 0 and lib.lk_attention_paged_workspace(8, 1, 64, 4, 2, 64, 64, 0) == 0
    for args, match in (*shared, ({**long}, "workspace too small"), ({**long, "ws": 16, "size": need - 1}, "workspace too"),
                        ({**long, "size": need}, "workspace too"), ({**long, "ws": 8, "size": need}, "16-byte aligned"),
                        ({"seqs": 65537, "rows": 65537}, "up to 65536"), ({"hk": 3}, "multiple of the key heads"), ({"d": 200}, "d_qk"), ({"dv": 136}, "d_v"),
                        ({"scale": float("nan")}, "finite"), ({"scale": 3e38}, "finite"), ({"qs": 12}, "multiples of 8"),
                        ({"row": 1 << 24}, "2\\^24"), ({"rows": (1 << 31) - 1, "h": 32768}, "too many query rows")):
        with pytest.raises(RuntimeError, match=match):
            attention(**args)
    attention(rows=0)
    for bad in ((-1, 1, 64, 4, 2, 64, 64), (8, 0, 64, 4, 2, 64, 64), (8, 1, -1, 4, 2, 64, 64),
                (8, 1, 64, 3, 2, 64, 64), (8, 1, 64, 4, 2, 200, 64), (8, 1, 64, 4, 2, 64, 136)):
        assert lib.lk_attention_paged_workspace(*bad, 0) == -1


def _copy(src, dst, pages=8, pointer=16, stride=4096, size=4096, count=1, pairs=None):
    ints = [(ctypes.c_int32 * max(1, len(x)))(*x) for x in (src, dst)]
    _lib.call("lk_copy_pages", (ctypes.c_void_p * 1)(pointer), (ctypes.c_int64 * 1)(stride),
              (ctypes.c_int64 * 1)(size), count, *ints, len(src) if pairs is None else pairs, pages, None, None)


def test_copies_are_refused_that_depend_on_each_other(lib):
    for src, dst, match in (([0, 1], [2, 2], "page 2 is written twice"), ([0, 2], [2, 3], "page 2 is both"),
                            ([0, 1], [1, 0], "both read and written"), ([8], [1], "pair 0 copies page 8 to 1"),
                            ([0, 1], [1, -1], "pair 0|pair 1"), ([5, 0, 1], [0, 1, 2], "both read"),
                            (list(range(300)), [700 - i // 2 for i in range(300)], "written twice")):
        with pytest.raises(RuntimeError, match=match):
            _copy(src, dst, pages=1000 if len(src) > 9 else 8)
    for kw, match in (({"pointer": None}, "null"), ({"pointer": 8}, "16-byte"), ({"size": 8}, "16 bytes"),
                      ({"stride": 2048}, "must not overlap"), ({"size": 1 << 31, "stride": 1 << 31}, "2\\^31"),
                      ({"pages": -1}, "0 .. 2"), ({"pairs": -1}, "0 .. 2")):
        with pytest.raises(RuntimeError, match=match):
            _copy([0], [1], **kw)
    _copy([], [])
    _copy([0], [1], count=0)


def test_the_oracles_forms_agree(rng):
    """Pages gathered token by token, and a rotation as a product of complex numbers."""
    table = np.array([[3, 0, -1], [1, 9, 2]], dtype=np.int32)
    got = P.places(table, [20, 40], 16, 4, 5, np.array([0, 2, 4]))
    assert got.tolist() == [[0, 18, 0, 2], [0, 19, 0, 3], [1, 38, 2, 6], [1, 39, 2, 7], [-1, -1, -1, -1]]
    assert P.places(table, [1, 20], 16, 4, 4)[:, 1:].tolist() == [[-1, -1, -1], [0, 3, 0], [18, -1, -1], [19, -1, -1]]
    assert P.places(table, [0, 50], 16, 4, 2)[:, 1:].tolist() == [[-1, -1, -1], [49, -1, -1]]
    x, a = rng.normal(size=(3, 2, 16)), rng.uniform(0, 6, (9, 4))
    cs = np.concatenate((np.cos(a), np.sin(a)), 1)
    for interleaved in (False, True):
        y, _ = P.rotate(x, cs, np.array([2, 5, 99]), None, 0.0, 8, interleaved)
        z = x[..., 8::2] + 1j * x[..., 9::2] if interleaved else x[..., 8:12] + 1j * x[..., 12:]
        z = z * np.exp(1j * a[[2, 5, 8]])[:, None]
        w = y[..., 8::2] + 1j * y[..., 9::2] if interleaved else y[..., 8:12] + 1j * y[..., 12:]
        assert np.allclose(z, w, rtol=1e-12) and np.array_equal(y[..., :8], x[..., :8])
    kp, vp = rng.normal(size=(4, 16, 1, 8)), rng.normal(size=(4, 16, 1, 4))
    q = rng.normal(size=(2, 2, 8))
    out, _, _, keys = P.attention_paged(q, kp, vp, table, [20, 0], 0.3, np.array([0, 1, 2]))
    k = np.concatenate((kp[3], kp[0, :4]))[:, 0]
    v = np.concatenate((vp[3], vp[0, :4]))[:, 0]
    p = np.exp(0.3 * (k @ q[0].T))
    assert keys == 20 and np.allclose(out[0], (p / p.sum(0)).T @ v) and not out[1].any()
