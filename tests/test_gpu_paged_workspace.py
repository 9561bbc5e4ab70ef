"""What attention on pages reads from its workspace and did not write in the same call."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .test_gpu_paged import DEV, _require_gpu, _t

pytestmark = pytest.mark.gpu

_ = _require_gpu  # fixture


def test_tiles_of_an_earlier_call_lead_nowhere():
    """A call whose offsets are out of order (its results are left open) can count tiles in runs
    that no block notes, and finds what an earlier call of other heads left there: the rows behind
    the output stay as they are."""
    from local_kimi_amd import _lib

    rows, n, d, page_rows, width = 640, 640, 64, 16, 128
    stream = torch.cuda.current_stream().cuda_stream
    k = torch.randn((width, page_rows, 1, d), device=DEV).bfloat16()
    table = torch.arange(width, dtype=torch.int32, device=DEV).repeat(n, 1)
    capacity = width * page_rows
    need = max(_lib.query("lk_attention_paged_workspace", rows, n, capacity, h, 1, d, d, 1) for h in (17, 4))
    ws = torch.zeros(need, dtype=torch.uint8, device=DEV)

    def call(heads, lengths, cu):
        q = torch.randn((rows, heads, d), device=DEV).bfloat16()
        out = torch.full((rows + 8, heads, d), 7.0, device=DEV).bfloat16()
        lengths, cu = _t(np.array(lengths), torch.int32), _t(np.array(cu), torch.int32)
        _lib.call("lk_attention_paged", q.data_ptr(), k.data_ptr(), k.data_ptr(), out.data_ptr(),
                  table.data_ptr(), lengths.data_ptr(), cu.data_ptr(), n, rows, heads, 1, d, d,
                  heads * d, d, width, page_rows, width, width, page_rows * d, d, d,
                  page_rows * d, d, d, 0.125, 2, ws.data_ptr(), need, stream)
        torch.cuda.synchronize()
        return out

    # single tokens of 17 heads: the one in runs is row 636, its tile the first
    lengths = [1] * n
    lengths[636] = 2000
    out = call(17, lengths, range(n + 1))
    assert bool((out[rows:] == 7).all()) and bool(out[:rows].isfinite().all())
    # every other sequence is all rows: more tiles than the call has blocks, those of the last
    # long sequence in runs; four heads a tile, so that 17 rows are five tokens
    lengths = [0] * n
    lengths[638] = 2000
    out = call(4, lengths, [0, rows] * (n // 2) + [0])
    assert bool((out[rows:] == 7).all())
