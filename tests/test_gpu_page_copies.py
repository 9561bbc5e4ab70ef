"""Copies of pages whose lists name a page with itself: such a pair does nothing, also where
another pair writes the page."""

from __future__ import annotations

import pytest
import torch

from .test_gpu_paged import DEV, _require_gpu

pytestmark = pytest.mark.gpu

_ = _require_gpu  # fixture


@pytest.mark.parametrize("values", [8, 1024, 64 * 1024])  # a page: in one block with others, of one block, of many
@pytest.mark.parametrize("others", [0, 300])                # the lists as arguments, and uploaded
@pytest.mark.parametrize("self_first", [False, True])
def test_a_page_with_itself_does_nothing(values, others, self_first):
    from local_kimi_amd.kernels import copy_pages

    pages = 8 + 2 * others
    t = torch.randint(0, 1 << 30, (pages, values), device=DEV, dtype=torch.int32)
    u = torch.randn((pages, 16), device=DEV)
    src, dst = [3, 1, 6], [3, 3, 6]
    if not self_first:
        src, dst = src[::-1], dst[::-1]
    src, dst = src + list(range(8, 8 + others)), dst + list(range(8 + others, pages))
    for _ in range(5):
        want = [x.clone() for x in (t, u)]
        for w in want:
            w[3] = w[1]
            w[8 + others:] = w[8:8 + others]
        copy_pages([t, u], src, dst)
        assert torch.equal(t, want[0]) and torch.equal(u, want[1])
        t[3] += 1
        u[3] += 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copy_pages([t, u], src, dst)
    for i in range(3):
        t.random_(0, 1 << 30)
        u.normal_()
        want = t.clone()
        want[3] = want[1]
        want[8 + others:] = want[8:8 + others]
        graph.replay()
        assert torch.equal(t, want), i
