"""Registers and LDS of the built prompt kernels: what lets two blocks of them
share a CU, and keeps their accumulators out of scratch memory."""

from __future__ import annotations

from .test_kernel_resources import _template_args, kernels

_ = kernels  # fixture


def _found(kernels, name):
    return {args: k for k in kernels if (args := _template_args(k[".name"], name)) is not None}


def test_attention_shares_a_cu(kernels):
    found = _found(kernels, "attention_kernel")
    assert len(found) == 6
    for args, k in found.items():
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, args
        assert k[".vgpr_count"] <= 256 and k[".group_segment_fixed_size"] <= 80 << 10, args


def test_chunk_kernels_keep_their_registers(kernels):
    prepare = _found(kernels, "chunk_prepare_kernel")
    assert len(prepare) == 6
    for args, k in prepare.items():
        assert k[".vgpr_spill_count"] == 0 and k[".vgpr_count"] <= 128, args
        assert k[".group_segment_fixed_size"] <= 80 << 10, args
    scan = _found(kernels, "chunk_scan_kernel")
    assert len(scan) == 12
    for args, k in scan.items():
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, args


def test_convolutions_and_steps_use_no_scratch_memory(kernels):
    for name, count in (("conv_prefill_kernel", 18), ("scan_serial_kernel", 9)):
        found = _found(kernels, name)
        assert len(found) == count
        assert not any(k[".private_segment_fixed_size"] for k in found.values()), name
