"""The state that decoding updates in place counts as written: a graph that saved it says so instead of using the new values."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from gdn2_tilelang_b200 import _cabi

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "python"], autouse=True)
def way(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_cabi.kernels(), "host", None)


@pytest.mark.parametrize("n", [1, 40])
def test_a_graph_that_saved_the_state(n):
    g = -torch.rand(2, n, 24, device="cuda")
    state, scale = torch.ones(2, 24, device="cuda"), torch.ones(24, device="cuda", requires_grad=True)
    y = (state * scale).sum()
    before = state._version
    gdn2.gated_recurrence_decode(torch.rand_like(g), g, None, state)
    assert state._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    whole = torch.ones(2, 48, device="cuda")           # a view counts for the tensor it is of
    part = whole.view(4, 24)[:2]
    gdn2.gated_recurrence_decode(torch.rand_like(g), g, None, part)
    assert whole._version == 1


def test_under_inference_mode():
    with torch.inference_mode():
        g = -torch.rand(2, 1, 24, device="cuda")
        state = torch.ones(2, 24, device="cuda")
        gdn2.gated_recurrence_decode(torch.rand_like(g), g, None, state)
    assert torch.isfinite(state).all()
