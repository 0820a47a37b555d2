"""A pre-activation that is not a number: its gradients say so, those of its neighbours do not."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("T", [20, 300])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_a_weight_that_is_not_a_number(T, act, dtype):
    """One element of w_gate: inner channel 7 of every token has no gate value, but a finite up projection."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    n = lambda *s: (torch.randn(*s, generator=gen, device="cuda") * 0.1).to(dtype)      # noqa: E731
    x, wg, wu, wd, dy = n(T, 72), n(40, 72), n(40, 72), n(24, 40), n(T, 24)
    wg[7, 3] = float("nan")
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    y = gdn2.gated_feed_forward(*leaves, act)
    dx, dwg, dwu, dwd = torch.autograd.grad(y, leaves, dy)
    assert torch.isnan(y).all() and torch.isnan(dx).all()
    assert torch.isnan(dwg[7]).all() and torch.isnan(dwu[7]).all() and torch.isnan(dwd[:, 7]).all()
    others = [i for i in range(40) if i != 7]
    assert torch.isfinite(dwg[others]).all() and torch.isfinite(dwu[others]).all() and torch.isfinite(dwd[:, others]).all()
