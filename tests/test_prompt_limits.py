"""Limits and rules of the prompt operators at the C ABI: all on the host, before any
launch, so they run without a GPU (no pointer here is dereferenced)."""

from __future__ import annotations

import pytest

from local_kimi_amd import _lib


@pytest.fixture(scope="module", autouse=True)
def _require_lib():
    if not _lib.is_built():
        pytest.skip("library not built; run python -m local_kimi_amd._build")


def _conv(tokens, channels, sequences=1):
    _lib.call("lk_kda_short_conv_prefill", *([16] * 15), None, sequences, tokens, channels, channels,
              2, 2, None)


def _scan(sequences, tokens, heads, d_k, d_v, workspace=None, size=0):
    _lib.call("lk_kda_prefill", *([16] * 8), None, sequences, tokens, heads, d_k, d_v, 1.0, 0,
              workspace, size, None)


def _attention(sequences, rows_q, rows_k, heads, kv_heads, d, workspace=None, size=0):
    _lib.call("lk_attention_prefill", 16, 16, 16, 16, None, None, sequences, rows_q, rows_k, heads,
              kv_heads, d, d, heads * d, d, kv_heads * d, d, kv_heads * d, d, 1.0, 2, workspace, size,
              None)


def test_grids_of_2_to_the_32_threads_are_refused():
    """2^26 tiles of 128 threads; 2^23 x 4 heads x 4 column blocks of 256; 2^24 blocks
    of 256."""
    with pytest.raises(RuntimeError, match="too many tokens and channels"):
        _conv(1 << 30, 8)
    with pytest.raises(RuntimeError, match="too many sequences x heads"):
        _scan(1 << 23, 1 << 23, 4, 64, 64)
    with _lib.forced_path("kda_prefill", "chunks"), \
            pytest.raises(RuntimeError, match="too many sequences x heads"):
        _scan(1 << 23, 1 << 23, 4, 64, 64, 16, 1 << 40)
    with pytest.raises(RuntimeError, match="too many query rows and heads"):
        _attention(1, 1 << 29, 1 << 29, 4, 2, 64)
