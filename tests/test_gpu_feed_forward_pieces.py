"""The gated gradient's epilogue where every warp works through many pieces: the same bits in every call, right ones in the first."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from tests import ffn_oracle as orc
from tests.test_gpu_feed_forward import BF, F16, NAMES, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("down", [True, False], ids=["with_dw_down", "without"])
@pytest.mark.parametrize("T,hid,inn,dtype", [(3100, 520, 4100, BF), (2050, 256, 5632, F16)])
def test_many_tiles_of_a_pair(T, hid, inn, dtype, act, down):
    """221 and 198 tiles on 74 pairs: three rounds, in which the last piece of a tile is followed by the first of the next. Without
    the gradient of w_down a third of the stores is left out, which changes what the loads wait behind."""
    x, wg, wu, wd, dy = make(T, hid, inn, dtype)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)][:4 if down else 3]
    call = lambda: torch.autograd.grad(gdn2.gated_feed_forward(*(leaves + [wd])[:4], act), leaves, dy)      # noqa: E731
    first = call()
    want = orc.evaluate(x, wg, wu, wd, act, dy)
    for name, g in zip(NAMES, first):
        orc.assert_within(g, *want[name], name)
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(200):
        for a, b in zip(call(), first):
            differ += (a != b).sum()
    assert int(differ) == 0
