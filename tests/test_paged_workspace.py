"""The workspace of attention on pages, as documented; no launch, so it runs without a GPU."""

from __future__ import annotations

import pytest

from local_kimi_amd import _lib


@pytest.mark.parametrize("rows,sequences,h,hk,packed,units", [
    (64, 64, 32, 8, False, 1), (64, 64, 16, 1, False, 1),          # up to 16 rows x heads a pack
    (64, 64, 32, 1, False, 2), (512, 64, 32, 8, False, 2), (64, 64, 34, 1, False, 2),   # up to 32
    (576, 64, 32, 8, False, 8), (64, 64, 32, 8, True, 8), (4, 2, 32, 8, True, 1), (64, 64, 37, 1, False, 1)])
def test_workspace_by_the_rows_of_a_pack(rows, sequences, h, hk, packed, units):
    if not _lib.is_built():
        pytest.skip("library not built; run python -m local_kimi_amd._build")
    lib = _lib.load()
    for d_v, dv in ((128, 128), (64, 64)):
        got = lib.lk_attention_paged_workspace(rows, sequences, 8192, h, hk, d_v, d_v, packed)
        sums = 2 * 1024 * units * 16 * (dv + 2) * 4  # 2048 runs of 16-row units, their sums and maxima in fp32
        assert sums <= got <= sums + (1 << 16)
        # from 256 sequences on 16 bytes a sequence more
        n = 1000 * rows // sequences
        more = lib.lk_attention_paged_workspace(n, 1000, 8192, h, hk, d_v, d_v, False)
        few = lib.lk_attention_paged_workspace(n // 1000, 1, 8192, h, hk, d_v, d_v, False)
        assert 16 * 1001 <= more - few < 16 * 1001 + 256
    assert lib.lk_attention_paged_workspace(rows, sequences, 256, h, hk, 64, 64, packed) == 0  # one run at the most
