"""Full attention on a cache that is kept in pages, on HIP.

What a full attention layer (engine/klinear/attention.py) does with its projected
queries, keys and values where the earlier tokens' keys and values are cached:
``qk_norm_rope`` (norm of each head and position rotation), ``qk_norm_rope_append``
(the same, with the keys and values written to the cache), ``paged_append`` (the write
alone), ``attention_paged`` (new tokens, one or many a sequence, on the cache) and
``copy_pages``. ``local_kimi_amd.paged.PagedCache`` keeps the pages. Kernels:
``local_kimi_amd/csrc/paged_cache.hip`` and ``paged_attention.hip``; outputs and
workspaces come from the torch caching allocator and nothing synchronises, so the
calls can be captured in a HIP graph.

A cache is ``k_pages`` [pages, rows, H_kv, d_qk] and ``v_pages`` [pages, rows, H_kv,
d_v], views of any strides that are multiples of 16 bytes (a page may hold its heads
first), rows a multiple of 16. ``page_table`` [N, M] int32 names each sequence's pages
in order, ``lengths`` [N] counts its tokens, the call's new ones included, which are its
last; both are read on the device, so a captured graph takes other contents. Table
entries that name no page (-1, say) lead nowhere.
"""

from __future__ import annotations

import ctypes
import math
from collections.abc import Sequence

import torch

from .. import _lib
from . import w4a16 as _w
from .attention import ATTENTION_MAX_QK_DIM, ATTENTION_MAX_V_DIM, _rows
from .kda import _aligned, _offsets

HEAD_MAX_DIM = 256
PAGE_ROWS_STEP = 16

_DTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def rope_table(positions: int, rotary_dim: int, theta: float = 10000.0, *,
               device: torch.device | str | None = None) -> torch.Tensor:
    """cos, then sin, of the angles p * theta ** (-2 i / rotary_dim) of positions
    0 .. ``positions`` - 1: fp32 [positions, rotary_dim], computed in 64 bits. Any such
    table (scaled frequencies, say) goes into the operators."""
    if rotary_dim <= 0 or rotary_dim % 8:
        raise ValueError(f"the rotated width must be a positive multiple of 8, got {rotary_dim}")
    rate = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * rate
    return torch.cat((angle.cos(), angle.sin()), 1).float().to(device)


# ---------------------------------------------------------------------------
# checks


def _check_angles(cos_sin, d, rotary_offset, device) -> tuple[torch.Tensor, int]:
    if cos_sin.ndim != 2 or cos_sin.shape[0] == 0:
        raise ValueError("cos_sin must have shape [positions, rotary_dim]")
    if cos_sin.dtype != torch.float32:
        raise TypeError(f"cos_sin must be float32, got {cos_sin.dtype}")
    if cos_sin.device != device:
        raise ValueError("cos_sin must be on the inputs' device")
    rotary = cos_sin.shape[1]
    if rotary == 0 or rotary % 8 or rotary_offset % 8 or rotary_offset < 0 or rotary_offset + rotary > d:
        raise ValueError(f"the rotated slice [{rotary_offset}, {rotary_offset + rotary}) must lie "
                         f"within the head's {d} values, in multiples of 8")
    return _aligned(cos_sin), rotary


def _check_weights(q_weight, k_weight, d, device, eps):
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight must both be given, or neither")
    if not eps >= 0:
        raise ValueError("eps must be non-negative")
    if q_weight is None:
        return None, None, 0
    for w in (q_weight, k_weight):
        if w.ndim != 1 or w.shape[0] != d:
            raise ValueError(f"the norm weights must have shape [{d}]")
        if w.device != device:
            raise ValueError("norm weights must be on the inputs' device")
    if q_weight.dtype not in _DTYPE_CODES or k_weight.dtype != q_weight.dtype:
        raise TypeError("the norm weights must share one dtype: float32, float16 or bfloat16")
    return _aligned(q_weight), _aligned(k_weight), _DTYPE_CODES[q_weight.dtype]


def _check_heads(q, k, max_dim=HEAD_MAX_DIM):
    if q.ndim != 4 or k.ndim != 4:
        raise ValueError("queries and keys must have shape [batch, sequence, heads, head_dim]")
    if k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
        raise ValueError("queries and keys must agree in batch, sequence and head_dim")
    if k.dtype != q.dtype:
        raise TypeError("queries and keys must share one dtype")
    if k.device != q.device:
        raise ValueError("queries and keys must share one device")
    if q.shape[2] == 0 or k.shape[2] == 0 or q.shape[0] == 0:
        raise ValueError("batch and heads must be nonzero")
    d = q.shape[3]
    if d == 0 or d % 8 or d > max_dim:
        raise ValueError(f"head_dim must be a positive multiple of 8 up to {max_dim}, got {d}")


def _check_cache(k_pages, v_pages, page_table, lengths, kv_heads, d_qk, dtype, device):
    """(d_v, the strides of both, the table, the lengths) of a cache that fits."""
    if k_pages.ndim != 4 or v_pages.ndim != 4 or k_pages.shape[:3] != v_pages.shape[:3]:
        raise ValueError("k_pages and v_pages must have shape [pages, rows, kv_heads, head_dim]")
    pages, rows, heads, width = k_pages.shape
    d_v = v_pages.shape[3]
    if heads != kv_heads or width != d_qk:
        raise ValueError(f"the cache holds {heads} heads of {width}, the call has {kv_heads} of {d_qk}")
    if rows == 0 or rows % PAGE_ROWS_STEP or rows > 65536:
        raise ValueError(f"a page must have a multiple of {PAGE_ROWS_STEP} rows up to 65536, got {rows}")
    if k_pages.dtype != dtype or v_pages.dtype != dtype:
        raise TypeError("the cache must have the inputs' dtype")
    if page_table.ndim != 2 or lengths.ndim != 1 or lengths.shape[0] != page_table.shape[0]:
        raise ValueError("page_table must have shape [sequences, pages a sequence], lengths "
                         "[sequences]")
    if page_table.dtype != torch.int32 or lengths.dtype not in (torch.int32, torch.int64):
        raise TypeError("page_table must be int32, lengths int32 or int64")
    if any(t.device != device for t in (k_pages, v_pages, page_table, lengths)):
        raise ValueError("the cache, its table and the lengths must be on the inputs' device")
    strides = []
    for t in (k_pages, v_pages):
        if t.shape[3] > 1 and t.stride(3) != 1 or any(s % 8 or s < 0 for s in t.stride()[:3]) \
                or t.data_ptr() % 16:
            raise ValueError("cached heads must be dense, and pages, rows and heads on 16 bytes")
        strides += t.stride()[:3]
    n, width = page_table.shape
    if width > 1 and page_table.stride(1) != 1 or n > 1 and page_table.stride(0) < width:
        page_table = page_table.contiguous()
    if lengths.dtype == torch.int64:  # beyond int32 is beyond every table
        lengths = lengths.clamp(0, 2 ** 31 - 1).to(torch.int32)
    return d_v, strides, page_table, _w._c(lengths)


def _table_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


# ---------------------------------------------------------------------------
# norms, rotation, append


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, cos_sin: torch.Tensor, positions: torch.Tensor,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                 eps: float = 1e-6, *, rotary_offset: int = 0,
                 interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of each head of ``q`` [B, S, H, d] and ``k`` [B, S, H_kv, d] (without
    weights: none), then the rotation of values ``rotary_offset`` to + rotary_dim by
    ``cos_sin`` [P, rotary_dim] at ``positions`` [B, S] (int32 or int64, clamped to the
    table): value i with i + rotary_dim / 2, or with ``interleaved`` 2 i with 2 i + 1.

    float32, float16 or bfloat16; computed in fp32 and rounded once. d is a multiple of
    8 up to 256, rotary_dim and rotary_offset multiples of 8. Strided inputs (slices of a
    fused projection) are read in place where rows and heads start on 16 bytes. Returns
    dense (q, k)."""
    _check_heads(q, k)
    code = _DTYPE_CODES.get(q.dtype)
    if code is None:
        raise TypeError(f"queries and keys must be float32, float16 or bfloat16, got {q.dtype}")
    batch, rows, heads, d = q.shape
    cs, rotary = _check_angles(cos_sin, d, rotary_offset, q.device)
    qw, kw, wcode = _check_weights(q_weight, k_weight, d, q.device, eps)
    if tuple(positions.shape) != (batch, rows):
        raise ValueError("positions must have shape [batch, sequence]")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if positions.device != q.device:
        raise ValueError("positions must be on the inputs' device")
    if q.device.type != "cuda":
        raise ValueError("the HIP head kernels require CUDA tensors")
    q_out = q.new_empty(q.shape)
    k_out = k.new_empty(k.shape)
    if rows:
        qc, kc, at = _rows(q), _rows(k), _w._c(positions)
        with _w._on(q.device):
            _lib.call("lk_qk_norm_rope", qc.data_ptr(), kc.data_ptr(),
                      None if qw is None else qw.data_ptr(), None if kw is None else kw.data_ptr(),
                      cs.data_ptr(), at.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
                      batch * rows, heads, k.shape[2], d, qc.stride(1), qc.stride(2), kc.stride(1),
                      kc.stride(2), rotary, rotary_offset, int(interleaved), cs.shape[0],
                      int(at.dtype == torch.int64), eps, code, wcode, _w._stream(q.device))
    return q_out, k_out


def _append(q, k, v, k_pages, v_pages, page_table, lengths, cos_sin, q_weight, k_weight, eps,
            cu_seqlens, rotary_offset, interleaved):
    batch, rows, kv_heads, d = k.shape
    if v.ndim != 4 or v.shape[:3] != k.shape[:3]:
        raise ValueError("v must have shape [batch, sequence, kv_heads, d_v]")
    code = _DTYPE_CODES.get(k.dtype)
    if code not in (1, 2):
        raise TypeError(f"cached values must be float16 or bfloat16, got {k.dtype}")
    if v.dtype != k.dtype:
        raise TypeError("keys and values must share one dtype")
    if v.device != k.device:
        raise ValueError("keys and values must share one device")
    d_v, strides, table, lengths = _check_cache(k_pages, v_pages, page_table, lengths, kv_heads, d,
                                                k.dtype, k.device)
    if v.shape[3] != d_v or d_v == 0 or d_v % 8 or d_v > HEAD_MAX_DIM:
        raise ValueError(f"values must have the cache's width, a multiple of 8 up to {HEAD_MAX_DIM}")
    cs, rotary = (None, 0) if cos_sin is None else _check_angles(cos_sin, d, rotary_offset, k.device)
    qw, kw, wcode = _check_weights(q_weight, k_weight, d, k.device, eps)
    offsets, count = _offsets(cu_seqlens, batch, k.device)
    if count != table.shape[0]:
        raise ValueError(f"the table has {table.shape[0]} sequences, the call {count}")
    if k.device.type != "cuda":
        raise ValueError("the HIP cache kernels require CUDA tensors")
    q_out = None if q is None else q.new_empty(q.shape)
    if rows:
        qc, kc, vc = None if q is None else _rows(q), _rows(k), _rows(v)
        with _w._on(k.device):
            _lib.call("lk_paged_append", None if q is None else qc.data_ptr(), kc.data_ptr(),
                      vc.data_ptr(), None if qw is None else qw.data_ptr(),
                      None if kw is None else kw.data_ptr(), None if cs is None else cs.data_ptr(),
                      table.data_ptr(), lengths.data_ptr(),
                      None if offsets is None else offsets.data_ptr(),
                      None if q is None else q_out.data_ptr(), k_pages.data_ptr(),
                      v_pages.data_ptr(), count, batch * rows, 0 if q is None else q.shape[2],
                      kv_heads, d, d_v, 0 if q is None else qc.stride(1),
                      0 if q is None else qc.stride(2), kc.stride(1), kc.stride(2), vc.stride(1),
                      vc.stride(2), k_pages.shape[0], k_pages.shape[1], table.shape[1],
                      _table_stride(table), *strides, rotary, rotary_offset, int(interleaved),
                      0 if cs is None else cs.shape[0], eps, code, wcode, _w._stream(k.device))
    return q_out


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor,
                        v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                        cos_sin: torch.Tensor, q_weight: torch.Tensor | None = None,
                        k_weight: torch.Tensor | None = None, eps: float = 1e-6, *,
                        cu_seqlens: torch.Tensor | None = None, rotary_offset: int = 0,
                        interleaved: bool = False) -> torch.Tensor:
    """``qk_norm_rope`` of new tokens at their positions in their sequences, with the
    keys and ``v`` [B, S, H_kv, d_v] written to the cache; returns the queries.

    Token i of the n that the call has of sequence s is position ``lengths[s]`` - n + i.
    B sequences of S new tokens each, or with ``cu_seqlens`` [N + 1] (int32 or int64, on
    the device, from 0, not decreasing) one row of N packed ones. A token without a place
    (a position below 0, no page) is not written, and rotated as position 0 where that is
    below 0; rows behind the last sequence write nothing and return zeros. Two sequences'
    new tokens must not share a page: copy a forked sequence's last page first
    (``PagedCache.extend`` does)."""
    _check_heads(q, k)
    return _append(q, k, v, k_pages, v_pages, page_table, lengths, cos_sin, q_weight, k_weight, eps,
                   cu_seqlens, rotary_offset, interleaved)


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor, *,
                 cu_seqlens: torch.Tensor | None = None) -> None:
    """``k`` [B, S, H_kv, d_qk] and ``v`` [B, S, H_kv, d_v] written to the cache as they
    are (layers without rotation); places as in ``qk_norm_rope_append``."""
    _check_heads(k, k)
    _append(None, k, v, k_pages, v_pages, page_table, lengths, None, None, None, 0.0, cu_seqlens, 0,
            False)


# ---------------------------------------------------------------------------
# attention


def attention_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    page_table: torch.Tensor, lengths: torch.Tensor, *,
                    scale: float | None = None,
                    cu_seqlens: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of new tokens on a paged cache that holds their keys and values
    behind the earlier ones: ``softmax(scale * q k^T) v`` over the positions each sees.

    ``q`` [B, S, H, d_qk], float16 or bfloat16 like the cache; H a multiple of H_kv, d_qk
    a multiple of 8 up to 192, d_v up to 128. B sequences of S new tokens, or with
    ``cu_seqlens`` [N + 1] one row of N packed ones, single tokens and long pieces side by
    side. New token i of n sees positions 0 .. ``lengths[s]`` - n + i; one that sees none
    gets zeros, as do the rows behind the last sequence. Lengths are clamped to what the
    table's row can name; positions without a page read as zeros.

    Returns [B, S, H, d_v] in q's dtype. ``scale`` defaults to d_qk ** -0.5. Scores and
    sums are fp32; the probabilities are rounded to the inputs' dtype for their product
    with the values."""
    code = _DTYPE_CODES.get(q.dtype)
    if code not in (1, 2):
        raise TypeError(f"attention inputs must be float16 or bfloat16, got {q.dtype}")
    if q.ndim != 4:
        raise ValueError("q must have shape [batch, sequence, heads, head_dim]")
    batch, rows, heads, d_qk = q.shape
    kv_heads = k_pages.shape[2] if k_pages.ndim == 4 else 0
    if batch == 0 or heads == 0 or kv_heads == 0 or heads % kv_heads:
        raise ValueError("the query heads must be a positive multiple of the key heads")
    if d_qk == 0 or d_qk % 8 or d_qk > ATTENTION_MAX_QK_DIM:
        raise ValueError(f"d_qk must be a positive multiple of 8 up to {ATTENTION_MAX_QK_DIM}, "
                         f"got {d_qk}")
    d_v, strides, table, lengths = _check_cache(k_pages, v_pages, page_table, lengths, kv_heads,
                                                d_qk, q.dtype, q.device)
    if d_v == 0 or d_v % 8 or d_v > ATTENTION_MAX_V_DIM:
        raise ValueError(f"d_v must be a positive multiple of 8 up to {ATTENTION_MAX_V_DIM}, "
                         f"got {d_v}")
    offsets, count = _offsets(cu_seqlens, batch, q.device)
    if count != table.shape[0]:
        raise ValueError(f"the table has {table.shape[0]} sequences, the call {count}")
    scale = d_qk ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if q.device.type != "cuda":
        raise ValueError("the HIP attention kernel requires CUDA tensors")
    out = q.new_empty((batch, rows, heads, d_v))
    if rows == 0:
        return out
    qc = _rows(q)
    need = _lib.query("lk_attention_paged_workspace", batch * rows, count,
                      table.shape[1] * k_pages.shape[1], heads, kv_heads, d_qk, d_v)
    ws = _w.workspace(need, q.device) if need else None
    with _w._on(q.device):
        _lib.call("lk_attention_paged", qc.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                  out.data_ptr(), table.data_ptr(), lengths.data_ptr(),
                  None if offsets is None else offsets.data_ptr(), count, batch * rows, heads,
                  kv_heads, d_qk, d_v, qc.stride(1), qc.stride(2), k_pages.shape[0],
                  k_pages.shape[1], table.shape[1], _table_stride(table), *strides, scale, code,
                  None if ws is None else ws.data_ptr(), need, _w._stream(q.device))
    return out


# ---------------------------------------------------------------------------
# copies


def _page_bytes(t: torch.Tensor) -> int:
    """Bytes of one page where a page is dense in some order of its dimensions."""
    dims = sorted((s, n) for s, n in zip(t.stride()[1:], t.shape[1:]) if n != 1)
    size = 1
    for s, n in dims:
        if s != size:
            raise ValueError("the pages of a copied tensor must be dense")
        size *= n
    return size * t.element_size()


def copy_pages(tensors: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int]) -> None:
    """Page ``src[i]`` to page ``dst[i]`` (dimension 0) of every tensor: all layers' caches,
    in one launch per 192 pairs of 64 tensors.

    ``src`` and ``dst`` are sequences of integers or integer tensors on the host; a page is
    written once at most, and is no other pair's source (ValueError). A captured graph
    keeps the lists it was captured with. Pages must be dense, in any order of their
    dimensions, and multiples of 16 bytes."""
    tensors = list(tensors)
    a, b = (torch.as_tensor(x, dtype=torch.int64, device="cpu") if len(x) else
            torch.empty(0, dtype=torch.int64) for x in (src, dst))
    if a.ndim != 1 or a.shape != b.shape:
        raise ValueError("src and dst must be lists of one length")
    if not tensors:
        return
    pages, device = tensors[0].shape[0], tensors[0].device
    sizes = []
    for t in tensors:
        if t.ndim < 2 or t.shape[0] != pages:
            raise ValueError("copied tensors must have shape [pages, ...], all of one number of pages")
        if t.device != device:
            raise ValueError("copied tensors must share one device")
        sizes.append(_page_bytes(t))
        if sizes[-1] % 16 or t.data_ptr() % 16 or t.stride(0) * t.element_size() % 16:
            raise ValueError("pages must be multiples of 16 bytes, on 16 bytes")
        if pages > 1 and t.stride(0) * t.element_size() < sizes[-1]:
            raise ValueError("the pages of a copied tensor must not overlap")
    if device.type != "cuda":
        raise ValueError("the HIP copy requires CUDA tensors")
    n = a.shape[0]
    if n == 0:
        return
    if bool(((a < 0) | (a >= pages) | (b < 0) | (b >= pages)).any()):
        raise ValueError(f"page numbers must be in 0 .. {pages - 1}")
    a, b = a.to(torch.int32), b.to(torch.int32)
    count = len(tensors)
    pointers = (ctypes.c_void_p * count)(*(t.data_ptr() for t in tensors))
    steps = (ctypes.c_int64 * count)(*(max(t.stride(0) * t.element_size(), s)
                                       for t, s in zip(tensors, sizes)))
    bytes_ = (ctypes.c_int64 * count)(*sizes)
    with _w._on(device):
        _lib.call("lk_copy_pages", pointers, steps, bytes_, count, a.data_ptr(), b.data_ptr(), n,
                  pages, _w._stream(device))
