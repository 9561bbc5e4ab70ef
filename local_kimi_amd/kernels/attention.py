"""Causal softmax attention over whole prompts on HIP.

``attention_prefill`` is what a full attention layer (engine/klinear/attention.py)
does with its projected queries, keys and values: grouped heads, query and key
heads wider than the value heads, equal sequences or packed ones of different
lengths, with or without earlier keys before each sequence's own. One launch of
``local_kimi_amd/csrc/attention.hip`` (two where few queries face many keys); the
output and any workspace come from the torch caching allocator and nothing
synchronises, so the call can be captured in a HIP graph.
"""

from __future__ import annotations

import math

import torch

from .. import _lib
from . import w4a16 as _w
from .kda import _offsets

ATTENTION_MAX_QK_DIM = 192
ATTENTION_MAX_V_DIM = 128
_DTYPE_CODES = {torch.float16: 1, torch.bfloat16: 2}


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` [B, S, H, D] as the kernel addresses it, copied where its layout is
    another: rows one stride apart through the batch, dense heads' values,
    16-byte steps."""
    fits = ((t.shape[3] == 1 or t.stride(3) == 1) and
            (t.shape[0] == 1 or t.stride(0) == t.shape[1] * t.stride(1)) and
            t.stride(1) % 8 == 0 and t.stride(2) % 8 == 0 and t.stride(1) < 1 << 24 and
            t.data_ptr() % 16 == 0)
    return t if fits else t.clone(memory_format=torch.contiguous_format)


def attention_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                      scale: float | None = None, cu_seqlens: torch.Tensor | None = None,
                      cu_seqlens_k: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of prompts: ``softmax(scale * q k^T) v`` over the keys
    each query sees.

    ``q`` [B, S, H, d_qk], ``k`` [B, S_k, H_kv, d_qk], ``v`` [B, S_k, H_kv, d_v],
    all float16 or all bfloat16; H a multiple of H_kv, d_qk a multiple of 8 up to 192,
    d_v up to 128. The queries are the last S of the S_k positions: query i
    sees keys 0 .. i + S_k - S, and one that sees none gets zeros.

    With ``cu_seqlens`` [N + 1] (int32 or int64, on the device, from 0, not
    decreasing) B is one and the S rows hold N packed sequences, whose keys are the same rows of
    ``k`` and ``v``, or with ``cu_seqlens_k`` [N + 1] the rows that it gives.
    Offsets are clamped to the rows; output rows behind the last sequence are
    zero.

    Returns [B, S, H, d_v] in q's dtype. ``scale`` defaults to d_qk ** -0.5.
    Scores and sums are fp32; the probabilities are rounded to the inputs'
    dtype for their product with ``v``. Strided inputs (a head's slice of a
    fused projection, heads expanded from one) are read in place where rows and
    heads start on 16 bytes.
    """
    code = _DTYPE_CODES.get(q.dtype)
    if code is None:
        raise TypeError(f"attention inputs must be float16 or bfloat16, got {q.dtype}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must share one dtype")
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError("q, k and v must have shape [batch, sequence, heads, head_dim]")
    batch, rows, heads, d_qk = q.shape
    _, rows_k, kv_heads, d_v = v.shape
    if tuple(k.shape) != (batch, rows_k, kv_heads, d_qk) or v.shape[0] != batch:
        raise ValueError("k must have shape [batch, keys, kv_heads, d_qk] and v [batch, keys, "
                         "kv_heads, d_v]")
    if batch == 0 or heads == 0 or kv_heads == 0 or heads % kv_heads:
        raise ValueError("the query heads must be a positive multiple of the key heads")
    if d_qk == 0 or d_qk % 8 or d_qk > ATTENTION_MAX_QK_DIM:
        raise ValueError(f"d_qk must be a positive multiple of 8 up to {ATTENTION_MAX_QK_DIM}, "
                         f"got {d_qk}")
    if d_v == 0 or d_v % 8 or d_v > ATTENTION_MAX_V_DIM:
        raise ValueError(f"d_v must be a positive multiple of 8 up to {ATTENTION_MAX_V_DIM}, "
                         f"got {d_v}")
    if not (q.device == k.device == v.device):
        raise ValueError("attention inputs must share one device")
    if cu_seqlens is None and cu_seqlens_k is not None:
        raise ValueError("cu_seqlens_k needs cu_seqlens")
    offsets, count = _offsets(cu_seqlens, batch, q.device)
    offsets_k = offsets
    if cu_seqlens_k is not None:
        offsets_k, count_k = _offsets(cu_seqlens_k, batch, q.device, "cu_seqlens_k")
        if count_k != count:
            raise ValueError("cu_seqlens and cu_seqlens_k must have the same length")
    elif cu_seqlens is not None and rows_k != rows:
        raise ValueError("packed sequences with keys of other rows need cu_seqlens_k")
    scale = d_qk ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if q.device.type != "cuda":
        raise ValueError("the HIP attention kernel requires CUDA tensors")
    out = q.new_empty((batch, rows, heads, d_v))
    if rows == 0:
        return out
    qc, kc, vc = _rows(q), _rows(k), _rows(v)
    need = _lib.query("lk_attention_prefill_workspace", batch * rows, batch * rows_k, count, heads,
                      kv_heads, d_qk, d_v)
    ws = _w.workspace(need, q.device) if need else None
    with _w._on(q.device):
        _lib.call("lk_attention_prefill", qc.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                  out.data_ptr(), None if offsets is None else offsets.data_ptr(),
                  None if offsets_k is None else offsets_k.data_ptr(), count, batch * rows,
                  batch * rows_k, heads, kv_heads, d_qk, d_v, qc.stride(1), qc.stride(2),
                  kc.stride(1), kc.stride(2), vc.stride(1), vc.stride(2), scale, code,
                  None if ws is None else ws.data_ptr(), need, _w._stream(q.device))
    return out
