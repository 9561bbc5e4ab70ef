"""Registers and LDS of the built paged-cache kernels."""

from __future__ import annotations

from .test_kernel_resources import kernels
from .test_prompt_resources import _found

_ = kernels  # fixture


def test_paged_attention_shares_a_cu(kernels):
    """Two blocks a CU: up to 256 registers and 80 KB; no scratch memory."""
    found = _found(kernels, "paged_attend_kernel")
    assert len(found) == 6
    for args, k in found.items():
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, args
        assert k[".vgpr_count"] <= 256 and k[".group_segment_fixed_size"] <= 80 << 10, args


def test_joins_and_heads_use_no_scratch_memory(kernels):
    for name, count in (("paged_join_kernel", 4), ("head_rope_kernel", 54)):
        found = _found(kernels, name)
        assert len(found) == count, name
        for args, k in found.items():
            assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, (name, args)
