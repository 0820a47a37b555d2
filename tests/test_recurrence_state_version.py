"""The state that decoding updates in place counts as written (no GPU: the kernel is a stand-in)."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from gdn2_tilelang_b200 import _cabi


class Kernels:
    host = None

    def recurrence(self, v, g, w, state, offsets, in_place=False):
        with torch.no_grad():
            state.data.add_(1)                         # as a kernel does it: autograd does not see it
        return torch.zeros_like(v), state, None

    def maybe_check_device_status(self, device):
        pass


def test_a_graph_that_saved_the_state(monkeypatch):
    monkeypatch.setattr(_cabi, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(_cabi, "kernels", Kernels)
    state, scale = torch.ones(2, 8), torch.ones(8, requires_grad=True)
    y = (state * scale).sum()
    x = torch.zeros(2, 1, 8)
    gdn2.gated_recurrence_decode(x, x, None, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        gdn2.gated_recurrence_decode(x, x, None, torch.ones(2, 8))
