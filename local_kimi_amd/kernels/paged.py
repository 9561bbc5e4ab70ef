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

import math
from array import array
from collections.abc import Sequence

import torch

from .. import _lib
from . import w4a16 as _w
from .attention import ATTENTION_MAX_QK_DIM, ATTENTION_MAX_V_DIM
from .kda import _aligned, _offsets

HEAD_MAX_DIM = 256
PAGE_ROWS_STEP = 16

_COPY_PAIRS = 192  # that a launch has room for in its arguments
_ERR_ARGUMENT = 1

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


def _check_angles(cos_sin, d, rotary_offset, device) -> tuple[torch.Tensor, int, int]:
    """The table as the kernels read it, its positions and its width."""
    if not isinstance(cos_sin, torch.Tensor):
        raise TypeError(f"cos_sin must be a tensor, got {type(cos_sin).__name__}")
    shape = cos_sin.shape
    if len(shape) != 2 or shape[0] == 0:
        raise ValueError("cos_sin must have shape [positions, rotary_dim]")
    if cos_sin.dtype is not torch.float32:
        raise TypeError(f"cos_sin must be float32, got {cos_sin.dtype}")
    if cos_sin.device != device:
        raise ValueError("cos_sin must be on the inputs' device")
    rows, rotary = shape
    if rotary == 0 or rotary % 8 or rotary_offset % 8 or rotary_offset < 0 or rotary_offset + rotary > d:
        raise ValueError(f"the rotated slice [{rotary_offset}, {rotary_offset + rotary}) must lie "
                         f"within the head's {d} values, in multiples of 8")
    return _aligned(cos_sin), rows, rotary


def _check_weights(q_weight, k_weight, d, device, eps):
    if not eps >= 0:
        raise ValueError("eps must be non-negative")
    if q_weight is None and k_weight is None:
        return None, None, 0
    if q_weight is None or k_weight is None:
        raise ValueError("q_weight and k_weight must both be given, or neither")
    for w in (q_weight, k_weight):
        if w.shape != (d,):
            raise ValueError(f"the norm weights must have shape [{d}]")
        if w.device != device:
            raise ValueError("norm weights must be on the inputs' device")
    code = _DTYPE_CODES.get(q_weight.dtype)
    if code is None or k_weight.dtype != q_weight.dtype:
        raise TypeError("the norm weights must share one dtype: float32, float16 or bfloat16")
    return _aligned(q_weight), _aligned(k_weight), code


def _check_heads(q, k):
    """(batch, sequence, query heads, key heads, head_dim, dtype, device)."""
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4:
        raise ValueError("queries and keys must have shape [batch, sequence, heads, head_dim]")
    batch, rows, heads, d = qs
    kbatch, krows, kv_heads, kd = ks
    if kbatch != batch or krows != rows or kd != d:
        raise ValueError("queries and keys must agree in batch, sequence and head_dim")
    dtype, device = q.dtype, q.device
    if k.dtype is not dtype:
        raise TypeError("queries and keys must share one dtype")
    if k.device != device:
        raise ValueError("queries and keys must share one device")
    if heads == 0 or kv_heads == 0 or batch == 0:
        raise ValueError("batch and heads must be nonzero")
    if d == 0 or d % 8 or d > HEAD_MAX_DIM:
        raise ValueError(f"head_dim must be a positive multiple of 8 up to {HEAD_MAX_DIM}, got {d}")
    return batch, rows, heads, kv_heads, d, dtype, device


def _check_cache(k_pages, v_pages, page_table, lengths, kv_heads, d_qk, dtype, device):
    """(d_v, table, lengths, [pages, rows, the table's width and stride, and the strides of
    keys' and values' pages, rows and heads]) of a cache that fits."""
    ks, vs = k_pages.shape, v_pages.shape
    if len(ks) != 4 or len(vs) != 4 or ks[:3] != vs[:3]:
        raise ValueError("k_pages and v_pages must have shape [pages, rows, kv_heads, head_dim]")
    pages, rows, heads, width = ks
    d_v = vs[3]
    if heads != kv_heads or width != d_qk:
        raise ValueError(f"the cache holds {heads} heads of {width}, the call has {kv_heads} of {d_qk}")
    if rows == 0 or rows % PAGE_ROWS_STEP or rows > 65536:
        raise ValueError(f"a page must have a multiple of {PAGE_ROWS_STEP} rows up to 65536, got {rows}")
    if k_pages.dtype is not dtype or v_pages.dtype is not dtype:
        raise TypeError("the cache must have the inputs' dtype")
    ts, ls = page_table.shape, lengths.shape
    if len(ts) != 2 or len(ls) != 1 or ls[0] != ts[0]:
        raise ValueError("page_table must have shape [sequences, pages a sequence], lengths "
                         "[sequences]")
    lengths_type = lengths.dtype
    if page_table.dtype is not torch.int32 or lengths_type not in (torch.int32, torch.int64):
        raise TypeError("page_table must be int32, lengths int32 or int64")
    if k_pages.device != device or v_pages.device != device or page_table.device != device \
            or lengths.device != device:
        raise ValueError("the cache, its table and the lengths must be on the inputs' device")
    a, b, c, x = k_pages.stride()
    e, f, g, y = v_pages.stride()
    if x != 1 and width > 1 or y != 1 and d_v > 1 or (a | b | c | e | f | g) % 8 \
            or min(a, b, c, e, f, g) < 0 or (k_pages.data_ptr() | v_pages.data_ptr()) % 16:
        raise ValueError("cached heads must be dense, and pages, rows and heads on 16 bytes")
    n, width = ts
    step, one = page_table.stride()
    if width > 1 and one != 1 or n > 1 and step < width:
        page_table, step = page_table.contiguous(), width
    if lengths_type is torch.int64:  # beyond int32 is beyond every table
        lengths = lengths.clamp(0, 2 ** 31 - 1).to(torch.int32)
    return (d_v, page_table, _w._c(lengths),
            (pages, rows, width, step if n > 1 else width, a, b, c, e, f, g))


def _heads_of(t: torch.Tensor, batch: int, rows: int) -> tuple[torch.Tensor, int, int]:
    """``t`` [batch, rows, heads, d] as the kernels address it, copied where its layout is
    another, and the strides of its rows and heads."""
    a, b, c, one = t.stride()
    if rows == 1:  # (a token of each sequence: any step between them)
        b = a
    if one == 1 and (batch == 1 or a == rows * b) and (b | c) % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, b, c
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride(1), t.stride(2)


def _pointer(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


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
    batch, rows, heads, kv_heads, d, dtype, device = _check_heads(q, k)
    code = _DTYPE_CODES.get(dtype)
    if code is None:
        raise TypeError(f"queries and keys must be float32, float16 or bfloat16, got {dtype}")
    cs, table_rows, rotary = _check_angles(cos_sin, d, rotary_offset, device)
    qw, kw, wcode = _check_weights(q_weight, k_weight, d, device, eps)
    if positions.shape != (batch, rows):
        raise ValueError("positions must have shape [batch, sequence]")
    at_type = positions.dtype
    if at_type is not torch.int32 and at_type is not torch.int64:
        raise TypeError(f"positions must be int32 or int64, got {at_type}")
    if positions.device != device:
        raise ValueError("positions must be on the inputs' device")
    if device.type != "cuda":
        raise ValueError("the HIP head kernels require CUDA tensors")
    q_out = torch.empty((batch, rows, heads, d), dtype=dtype, device=device)
    k_out = torch.empty((batch, rows, kv_heads, d), dtype=dtype, device=device)
    if rows:
        (q, q_row, q_head), (k, k_row, k_head) = _heads_of(q, batch, rows), _heads_of(k, batch, rows)
        at = _w._c(positions)
        with _w._on(device):
            _lib.call("lk_qk_norm_rope", q.data_ptr(), k.data_ptr(), _pointer(qw), _pointer(kw),
                      cs.data_ptr(), at.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
                      batch * rows, heads, kv_heads, d, q_row, q_head, k_row, k_head, rotary,
                      rotary_offset, bool(interleaved), table_rows, at_type is torch.int64, eps,
                      code, wcode, _w._stream(device))
    return q_out, k_out


def _append(q, heads, k, v, batch, rows, kv_heads, d, dtype, device, k_pages, v_pages, page_table,
            lengths, cos_sin, q_weight, k_weight, eps, cu_seqlens, rotary_offset, interleaved):
    vs = v.shape
    if len(vs) != 4 or vs[:3] != (batch, rows, kv_heads):
        raise ValueError("v must have shape [batch, sequence, kv_heads, d_v]")
    code = _DTYPE_CODES.get(dtype)
    if code != 1 and code != 2:
        raise TypeError(f"cached values must be float16 or bfloat16, got {dtype}")
    if v.dtype is not dtype:
        raise TypeError("keys and values must share one dtype")
    if v.device != device:
        raise ValueError("keys and values must share one device")
    d_v, table, lengths, layout = _check_cache(k_pages, v_pages, page_table, lengths, kv_heads, d,
                                               dtype, device)
    if vs[3] != d_v or d_v == 0 or d_v % 8 or d_v > HEAD_MAX_DIM:
        raise ValueError(f"values must have the cache's width, a multiple of 8 up to {HEAD_MAX_DIM}")
    cs, table_rows, rotary = (None, 0, 0) if cos_sin is None else \
        _check_angles(cos_sin, d, rotary_offset, device)
    qw, kw, wcode = _check_weights(q_weight, k_weight, d, device, eps)
    offsets, count = _offsets(cu_seqlens, batch, device)
    if count != table.shape[0]:
        raise ValueError(f"the table has {table.shape[0]} sequences, the call {count}")
    if device.type != "cuda":
        raise ValueError("the HIP cache kernels require CUDA tensors")
    q_out = torch.empty((batch, rows, heads, d), dtype=dtype, device=device) if heads else None
    if rows:
        q, q_row, q_head = _heads_of(q, batch, rows) if heads else (None, 0, 0)
        (k, k_row, k_head), (v, v_row, v_head) = _heads_of(k, batch, rows), _heads_of(v, batch, rows)
        with _w._on(device):
            _lib.call("lk_paged_append", _pointer(q), k.data_ptr(), v.data_ptr(), _pointer(qw),
                      _pointer(kw), _pointer(cs), table.data_ptr(), lengths.data_ptr(),
                      _pointer(offsets), _pointer(q_out), k_pages.data_ptr(), v_pages.data_ptr(),
                      count, batch * rows, heads, kv_heads, d, d_v, q_row, q_head, k_row, k_head,
                      v_row, v_head, *layout, rotary, rotary_offset, bool(interleaved), table_rows,
                      eps, code, wcode, _w._stream(device))
    return q_out


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor,
                        v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                        cos_sin: torch.Tensor | None, q_weight: torch.Tensor | None = None,
                        k_weight: torch.Tensor | None = None, eps: float = 1e-6, *,
                        cu_seqlens: torch.Tensor | None = None, rotary_offset: int = 0,
                        interleaved: bool = False) -> torch.Tensor:
    """``qk_norm_rope`` of new tokens at their positions in their sequences, with the
    keys and ``v`` [B, S, H_kv, d_v] written to the cache; returns the queries. With
    ``cos_sin`` None nothing is rotated.

    Token i of the n that the call has of sequence s is position ``lengths[s]`` - n + i.
    B sequences of S new tokens each, or with ``cu_seqlens`` [N + 1] (int32 or int64, on
    the device, from 0, not decreasing) one row of N packed ones. A token without a place
    (a position below 0 or beyond the table, no page) is not written; positions below 0 are
    rotated as 0. Rows behind the last sequence write nothing and return zeros. Two sequences'
    new tokens must not share a page: copy a forked sequence's last page first
    (``PagedCache.extend`` does). The cache's places must not overlap."""
    batch, rows, heads, kv_heads, d, dtype, device = _check_heads(q, k)
    return _append(q, heads, k, v, batch, rows, kv_heads, d, dtype, device, k_pages, v_pages,
                   page_table, lengths, cos_sin, q_weight, k_weight, eps, cu_seqlens, rotary_offset,
                   interleaved)


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor, *,
                 cu_seqlens: torch.Tensor | None = None) -> None:
    """``k`` [B, S, H_kv, d_qk] and ``v`` [B, S, H_kv, d_v] written to the cache as they
    are (layers without rotation); places as in ``qk_norm_rope_append``."""
    batch, rows, kv_heads, _, d, dtype, device = _check_heads(k, k)
    _append(None, 0, k, v, batch, rows, kv_heads, d, dtype, device, k_pages, v_pages, page_table,
            lengths, None, None, None, 0.0, cu_seqlens, 0, False)


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
    side. New token i of n sees positions 0 .. ``lengths[s]`` - n + i, of those that the table's
    row can name; one that sees none gets zeros, as do the rows behind the last sequence.
    Positions within the table that have no page read as zeros.

    Returns [B, S, H, d_v] in q's dtype. ``scale`` defaults to d_qk ** -0.5. Scores and
    sums are fp32; the probabilities are rounded to the inputs' dtype for their product
    with the values."""
    dtype, shape, device = q.dtype, q.shape, q.device
    code = _DTYPE_CODES.get(dtype)
    if code != 1 and code != 2:
        raise TypeError(f"attention inputs must be float16 or bfloat16, got {dtype}")
    if len(shape) != 4:
        raise ValueError("q must have shape [batch, sequence, heads, head_dim]")
    batch, rows, heads, d_qk = shape
    kv_heads = k_pages.shape[2] if k_pages.ndim == 4 else 0
    if batch == 0 or heads == 0 or kv_heads == 0 or heads % kv_heads:
        raise ValueError("the query heads must be a positive multiple of the key heads")
    if d_qk == 0 or d_qk % 8 or d_qk > ATTENTION_MAX_QK_DIM:
        raise ValueError(f"d_qk must be a positive multiple of 8 up to {ATTENTION_MAX_QK_DIM}, "
                         f"got {d_qk}")
    d_v, table, lengths, layout = _check_cache(k_pages, v_pages, page_table, lengths, kv_heads, d_qk,
                                               dtype, device)
    if d_v == 0 or d_v % 8 or d_v > ATTENTION_MAX_V_DIM:
        raise ValueError(f"d_v must be a positive multiple of 8 up to {ATTENTION_MAX_V_DIM}, "
                         f"got {d_v}")
    offsets, count = _offsets(cu_seqlens, batch, device)
    if count != table.shape[0]:
        raise ValueError(f"the table has {table.shape[0]} sequences, the call {count}")
    scale = d_qk ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if device.type != "cuda":
        raise ValueError("the HIP attention kernel requires CUDA tensors")
    out = torch.empty((batch, rows, heads, d_v), dtype=dtype, device=device)
    if rows == 0:
        return out
    q, q_row, q_head = _heads_of(q, batch, rows)
    need = _lib.query("lk_attention_paged_workspace", batch * rows, count, layout[1] * layout[2],
                      heads, kv_heads, d_qk, d_v, offsets is not None)
    ws = _w.workspace(need, device) if need else None
    with _w._on(device):
        _lib.call("lk_attention_paged", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                  out.data_ptr(), table.data_ptr(), lengths.data_ptr(), _pointer(offsets), count,
                  batch * rows, heads, kv_heads, d_qk, d_v, q_row, q_head, *layout, scale, code,
                  _pointer(ws), need, _w._stream(device))
    return out


# ---------------------------------------------------------------------------
# copies


def _page_layout(shape, strides, size: int) -> tuple[int, int]:
    """Bytes from a page to the next and of one page, which is dense in some order of its
    dimensions."""
    page = 1
    for step, n in sorted(x for x in zip(strides[1:], shape[1:]) if x[1] != 1):
        if step != page:
            raise ValueError("the pages of a copied tensor must be dense")
        page *= n
    page, step = page * size, strides[0] * size
    if shape[0] > 1 and step < page:
        raise ValueError("the pages of a copied tensor must not overlap")
    step = max(step, page)
    if page % 16 or step % 16:
        raise ValueError("pages must be multiples of 16 bytes, on 16 bytes")
    return step, page


def _page_list(pages: Sequence[int] | torch.Tensor, what: str) -> array:
    if isinstance(pages, torch.Tensor):
        if pages.device.type != "cpu" or pages.ndim != 1 or pages.is_floating_point():
            raise ValueError(f"{what} must be a list of integers on the host")
        pages = pages.tolist()
    try:
        return array("i", pages)
    except OverflowError:
        raise ValueError(f"{what} has page numbers beyond 2^31 - 1") from None


def copy_pages(tensors: Sequence[torch.Tensor], src: Sequence[int] | torch.Tensor,
               dst: Sequence[int] | torch.Tensor) -> None:
    """Page ``src[i]`` to page ``dst[i]`` (dimension 0) of every tensor: all layers' caches,
    in one launch for 64 tensors (while a graph is captured: and 192 pairs).

    ``src`` and ``dst`` are sequences of integers or integer tensors on the host; a page is
    written once at most, and is no other pair's source (ValueError); a pair of a page with
    itself does nothing. A captured graph keeps the lists it was captured with. Pages must be
    dense, in any order of their dimensions, and multiples of 16 bytes; the tensors must not
    overlap each other."""
    a, b = _page_list(src, "src"), _page_list(dst, "dst")
    if len(a) != len(b):
        raise ValueError("src and dst must be lists of one length")
    if not tensors:
        return
    pages, device = (tensors[0].shape or (0,))[0], tensors[0].device
    known: dict = {}  # most tensors are laid out alike
    pointers, steps, sizes = [], [], []
    for t in tensors:
        key = t.shape, t.stride(), t.dtype
        layout = known.get(key)
        if layout is None:
            if len(key[0]) < 2 or key[0][0] != pages:
                raise ValueError("copied tensors must have shape [pages, ...], all of one number of "
                                 "pages")
            layout = known[key] = _page_layout(key[0], key[1], t.element_size())
        if t.device != device:
            raise ValueError("copied tensors must share one device")
        pointers.append(t.data_ptr())
        if pointers[-1] % 16:
            raise ValueError("pages must be multiples of 16 bytes, on 16 bytes")
        steps.append(layout[0])
        sizes.append(layout[1])
    if device.type != "cuda":
        raise ValueError("the HIP copy requires CUDA tensors")
    if not a:
        return
    count, lists = len(a), None
    tables = [array("q", x) for x in (pointers, steps, sizes)]
    with _w._on(device):
        # (whether the stream that the launch goes to is captured: that of the tensors' device)
        if count > _COPY_PAIRS and not torch.cuda.is_current_stream_capturing():
            # from pinned memory of its own, so that the upload takes its turn on the stream
            lists = torch.frombuffer(a + b, dtype=torch.int32).pin_memory().to(device, non_blocking=True)
        status = _lib.load().lk_copy_pages(
            *(t.buffer_info()[0] for t in tables), len(pointers), a.buffer_info()[0],
            b.buffer_info()[0], count, pages, _pointer(lists), _w._stream(device))
    if status:
        message = _lib.load().lk_last_error().decode(errors="replace")
        raise (ValueError if status == _ERR_ARGUMENT else RuntimeError)(f"lk_copy_pages: {message}")
