"""Which stream a page copy asks about its capture; CPU only, the device and the library are stand-ins."""

from __future__ import annotations

import contextlib

import pytest
import torch

from local_kimi_amd.kernels import paged


class _Tensor:
    """A tensor of 1000 pages on a device that need not be there."""

    shape, dtype, device = torch.Size((1000, 4)), torch.float32, torch.device("cuda", 1)

    def stride(self):
        return 4, 1

    def element_size(self):
        return 4

    def data_ptr(self):
        return 4096


@pytest.mark.parametrize("pairs", [192, 193])
def test_the_capture_of_the_tensors_device_counts(monkeypatch, pairs):
    """The tensors' device is captured and is not the current one: the lists travel as arguments, for an
    upload would be recorded with memory that is free again at the replay."""
    current, calls = [0], []

    @contextlib.contextmanager
    def on(device):
        before, current[0] = current[0], device.index
        yield
        current[0] = before

    class Library:
        @staticmethod
        def lk_copy_pages(*args):
            calls.append(args)
            return 0

    monkeypatch.setattr(paged._w, "_on", on)
    monkeypatch.setattr(paged._w, "_stream", lambda device: 7)
    monkeypatch.setattr(paged._lib, "load", Library)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[0] == 1)
    monkeypatch.setattr(torch, "frombuffer", lambda *a, **k: pytest.fail("an upload within a capture"))
    paged.copy_pages([_Tensor()], list(range(pairs)), list(range(300, 300 + pairs)))
    assert len(calls) == 1 and calls[0][3] == 1 and calls[0][6:] == (pairs, 1000, None, 7) and current == [0]
