"""Operands that lie transposed in memory and have odd sizes: brought together first, then copied to aligned rows, all at once."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from gdn2_tilelang_b200 import _cabi
from tests import ffn_oracle as orc
from tests.test_gpu_feed_forward import BF, F16, NAMES, make

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "python"], autouse=True)
def way(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_cabi.kernels(), "host", None)


@pytest.mark.parametrize("T,hid,inn,out", [(5, 71, 133, 69), (130, 71, 133, 69), (300, 71, 71, 71), (257, 1001, 513, 255)])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_every_operand_transposed(T, hid, inn, out, dtype):
    plain = make(T, hid, inn, dtype, out, seed=T)
    want = orc.evaluate(*plain[:4], "silu", plain[4])
    leaves = [t.t().contiguous().t().requires_grad_() for t in plain[:4]]
    assert all(t.stride(0) == 1 for t in leaves)
    dy = plain[4].t().contiguous().t()
    for _ in range(5):
        with torch.no_grad():
            orc.assert_within(gdn2.gated_feed_forward(*leaves), *want["y"], "y")
        y = gdn2.gated_feed_forward(*leaves)
        orc.assert_within(y, *want["y"], "y")
        for name, g in zip(NAMES, torch.autograd.grad(y, leaves, dy)):
            orc.assert_within(g, *want[name], name)
