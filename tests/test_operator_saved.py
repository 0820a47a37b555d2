"""Tensors brought back by hooks as something else are refused before anything is launched (no GPU: the library is a stand-in)."""

from __future__ import annotations

import contextlib

import pytest
import torch

from gdn2_tilelang_b200 import _cabi

BF = torch.bfloat16


class Lib:
    """Sizes are answered, launches are not expected."""

    def gdn2_recurrence_marks(self, B, S, cu, sequences):
        return B * -(-S // 64)

    def gdn2_ffn_kept_bytes(self, tokens, stride):
        return 6 * tokens * stride


@pytest.fixture
def K(monkeypatch):
    k = _cabi.NativeKernels.__new__(_cabi.NativeKernels)
    k.lib, k.launches = Lib(), 0
    monkeypatch.setattr(_cabi, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(_cabi, "_on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(k, "_stream", lambda t: 0, raising=False)
    return k


CHANGES = {"type": lambda t: t.double() if t.is_floating_point() else t.int(), "shape": lambda t: t[:1] if t.shape[0] > 1 else t[..., :1],
           "device": lambda t: t.to("meta"), "rank": lambda t: t.unsqueeze(0)}


def refused(call, ins, change):
    for which in range(len(ins)):
        changed = [CHANGES[change](t) if i == which else t for i, t in enumerate(ins)]
        with pytest.raises(RuntimeError, match="came back from a hook"):
            call(*changed)
    with pytest.raises(AttributeError, match="gdn2_"):       # as it was saved, the call gets as far as the library
        call(*ins)


@pytest.mark.parametrize("change", CHANGES)
def test_recurrence(K, change):
    v, g, w, marks = torch.zeros(2, 70, 8, dtype=BF), torch.zeros(2, 70, 8), torch.zeros(2, 70, 8, dtype=BF), torch.zeros(4, 8)
    do, dfinal = torch.zeros(2, 70, 8, dtype=BF), torch.zeros(2, 8)
    refused(lambda v, g, w, marks: K.recurrence_backward(v, g, w, marks, do, dfinal, None, True), [v, g, w, marks], change)


@pytest.mark.parametrize("change", CHANGES)
def test_feed_forward(K, change):
    x, wg, wu, wd = (torch.zeros(*s, dtype=BF) for s in ((5, 8), (16, 8), (16, 8), (24, 16)))
    kept, dy = torch.zeros(6 * 5 * 16, dtype=torch.uint8), torch.zeros(5, 24, dtype=BF)
    refused(lambda *a: K.ffn_backward(*a, dy, "silu", True, True, True), [x, wg, wu, wd, kept], change)
