"""Operands that are brought together and then copied to aligned rows: what the copies read is alive when they are launched (no GPU)."""

from __future__ import annotations

import contextlib
import gc

import pytest
import torch

from gdn2_tilelang_b200 import _cabi

BF = torch.bfloat16


class Lib:
    def __init__(self):
        self.calls = 0

    def gdn2_align_rows(self, copies, n, stream):
        self.calls += 1
        live = {}
        for t in gc.get_objects():
            if type(t) is torch.Tensor and t.dtype == BF:
                live.setdefault(t.data_ptr(), []).append(tuple(t.shape))
        for c in copies:
            assert (c.rows, c.cols) in live.get(c.src, []), "a copy's source has been freed"
        return 0


@pytest.mark.parametrize("n", [1, 2, 4])
def test_sources_are_alive(n, monkeypatch):
    K = _cabi.NativeKernels.__new__(_cabi.NativeKernels)
    K.lib, K.launches = Lib(), 0
    monkeypatch.setattr(_cabi, "_on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(K, "_stream", lambda t: 0, raising=False)
    K.aligned_rows(*(torch.zeros(71, 9 + i, dtype=BF).t() for i in range(n)))       # columns apart, odd rows when brought together
    assert K.lib.calls == 1
