"""Limits and rules of the prompt operators at the C ABI: all on the host, before any
launch, so they run without a GPU (no pointer here is dereferenced)."""

from __future__ import annotations

import pytest

from local_kimi_amd import _lib

from .test_kernel_resources import kernels
from .test_prompt_resources import _found

_ = kernels  # fixture


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


def _attention(sequences, rows_q, rows_k, heads, kv_heads, d, workspace=None, size=0, scale=1.0):
    _lib.call("lk_attention_prefill", 16, 16, 16, 16, None, None, sequences, rows_q, rows_k, heads,
              kv_heads, d, d, heads * d, d, kv_heads * d, d, kv_heads * d, d, scale, 2, workspace,
              size, None)


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


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38, -3e38])
def test_scales_that_log2_e_takes_to_infinity_are_refused(scale):
    """Scores are scaled by scale * log2(e) in fp32: NaN for every result beyond it."""
    with pytest.raises(RuntimeError, match="scale must be finite"):
        _attention(1, 1, 1, 4, 2, 64, scale=scale)


@pytest.mark.parametrize("sequences,tokens,heads,d_k,d_v,chunks", [
    (1, 47, 4, 64, 64, False), (1, 48, 4, 64, 64, True), (3, 143, 4, 64, 64, False),
    (3, 144, 4, 64, 64, True), (1, 500, 4, 128, 64, True), (1, 500, 4, 129, 64, False),
    (1, 500, 4, 256, 64, False), (1, 500, 1 << 14, 16, (1 << 10) - 1, True),
    (1, 500, 1 << 14, 16, 1 << 10, False), (1, 0, 4, 64, 64, False)])
def test_the_form_that_a_scan_chooses(sequences, tokens, heads, d_k, d_v, chunks):
    """Chunks have a workspace, steps none: from 48 tokens a sequence on, up to d_k
    = 128, below 2^24 values a row."""
    size = _lib.query("lk_kda_prefill_workspace", sequences, tokens, heads, d_k, d_v)
    assert (size > 0) == chunks
    with _lib.forced_path("kda_prefill", "steps"):
        assert _lib.query("lk_kda_prefill_workspace", sequences, tokens, heads, d_k, d_v) == 0


def test_workspaces_a_byte_short_or_off_16_bytes_are_refused():
    need = _lib.query("lk_kda_prefill_workspace", 2, 500, 4, 64, 64)
    for size in (0, need - 1):
        with pytest.raises(RuntimeError, match="KDA prefill workspace too small"):
            _scan(2, 500, 4, 64, 64, 16, size)
    with pytest.raises(RuntimeError, match="KDA prefill workspace too small"):
        _scan(2, 500, 4, 64, 64, None, need)
    with pytest.raises(RuntimeError, match="workspace must be 16-byte aligned"):
        _scan(2, 500, 4, 64, 64, 8, need)
    need = _lib.query("lk_attention_prefill_workspace", 1, 5000, 1, 4, 2, 64, 64)
    assert need > 0
    for size in (0, need - 1):
        with pytest.raises(RuntimeError, match="attention workspace too small"):
            _attention(1, 1, 5000, 4, 2, 64, 16, size)
    with pytest.raises(RuntimeError, match="workspace must be 16-byte aligned"):
        _attention(1, 1, 5000, 4, 2, 64, 8, need)


def test_scalars_and_scratch_memory(kernels):
    """No kernel of a prompt has scratch memory; scalars that do not fit are kept in
    lanes of a vector register or two, as many as they are now."""
    limits = {"attention_kernel": 72, "attention_join_kernel": 0, "chunk_prepare_kernel": 8,
              "chunk_scan_kernel": 0, "scan_serial_kernel": 56, "conv_prefill_kernel": 0}
    for name, spills in limits.items():
        found = _found(kernels, name)
        assert found, name
        for args, k in found.items():
            assert k[".private_segment_fixed_size"] == 0 and k[".vgpr_spill_count"] == 0, (name, args)
            assert k[".sgpr_spill_count"] <= spills, (name, args)
