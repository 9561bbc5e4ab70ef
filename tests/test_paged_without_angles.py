"""Calls without a table of angles: an append that norms alone, a rotation that is refused."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from local_kimi_amd.kernels import qk_norm_rope, qk_norm_rope_append
from oracle import paged as P

from .test_gpu_paged import _close, _head_bound, _np

BF = torch.bfloat16


def test_a_rotation_without_angles_is_refused():
    q, k = torch.zeros(1, 6, 4, 64, dtype=BF), torch.zeros(1, 6, 2, 64, dtype=BF)
    at, w = torch.zeros(1, 6, dtype=torch.int32), torch.ones(64)
    for cos_sin, name in ((None, "NoneType"), (np.zeros((9, 64), np.float32), "ndarray")):
        with pytest.raises(TypeError, match=f"cos_sin must be a tensor, got {name}"):
            qk_norm_rope(q, k, cos_sin, at, w, w)
    pages = torch.zeros(5, 16, 2, 64, dtype=BF)
    with pytest.raises(TypeError, match="cos_sin must be a tensor, got list"):
        qk_norm_rope_append(q, k, k, pages, pages.clone(), torch.zeros(1, 3, dtype=torch.int32),
                            torch.zeros(1, dtype=torch.int32), [[1.0]])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm", [False, True])
def test_appends_without_a_rotation(dtype, norm):
    """The norm within its bound (test_gpu_paged.py: the mean of squares, its root and the products in
    fp32, one rounding; a call that rotates adds the squares in another order, so the two are not the
    same bit for bit), and without a norm the values as they are."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn((1, 21, n, d), generator=g, device="cuda").to(dtype) for n, d in ((6, 64), (2, 64), (2, 40)))
    w = [torch.rand(64, generator=g, device="cuda") if norm else None for _ in range(2)]
    table = torch.arange(4, dtype=torch.int32, device="cuda").reshape(2, 2)
    lengths, cu = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([30, 11], [0, 14, 21]))
    pages = [torch.full((4, 16, 2, d), 3.0, device="cuda", dtype=dtype) for d in (64, 40)]
    q_out = qk_norm_rope_append(q, k, v, *pages, table, lengths, None, *w, 1e-5, cu_seqlens=cu)
    k_pages, v_pages = pages
    assert torch.equal(v_pages[1, :14], v[0, :14]) and torch.equal(v_pages[2, 4:11], v[0, 14:])
    written = torch.zeros((4, 16), dtype=torch.bool, device="cuda")
    written[1, :14], written[2, 4:11] = True, True
    assert bool((k_pages[~written] == 3).all()) and bool((v_pages[~written] == 3).all())
    keys = torch.cat((k_pages[1, :14], k_pages[2, 4:11]))
    if not norm:
        assert torch.equal(q_out, q) and torch.equal(keys, k[0])
        return
    for x, got, weight in ((q, q_out, w[0]), (k, keys, w[1])):
        want, size = P.rotate(_np(x[0]), None, None, _np(weight), 1e-5)
        _close(got, want, _head_bound(want, size, 64, dtype))
