"""What a training step keeps of the two projections' sums (24 bits in a plane of 16 and one of 8) and what its gradients gain by it.

Bounds. The planes hold the float32 sums rounded to 15 bits behind the point: half a step is 2^-16 of the value, beside the float32
reduction's K 2^-24 of the terms' magnitudes. Whole numbers below 2^15 come back as they are.

In the 2-norm a rounding to nearest adds at most half / sqrt(3) of what it rounds (the error is uniform over a step, and a step is
largest against the value at the lower end of a binade); roundings are independent of one another and of the factors they are multiplied
by. With a and u in 24 bits every result has two of them behind it: h and y, da or du and dx or dw, h and dw_down. So
sqrt(2 / 3) half bounds all five. Dropping the lower planes would truncate a and u to 8 bits: a uniform error over a whole step,
2 half / sqrt(3) more for each of them."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from gdn2_tilelang_b200 import _cabi
from tests import ffn_oracle as orc
from tests.test_gpu_feed_forward import BF, F16, NAMES, make

pytestmark = pytest.mark.gpu


def kept_values(kept, T, inn):
    """The planes as float32 ``a, u [T, inn]``."""
    pitch = -(-inn // 16) * 16
    n = T * pitch
    upper = kept[:4 * n].view(torch.int16).view(2, T, pitch)[..., :inn].int() & 0xffff
    lower = kept[4 * n:6 * n].view(2, T, pitch)[..., :inn].int()
    return ((upper << 16) | (lower << 8)).view(torch.float32)


def keep(x, wg, wu, wd):
    K = _cabi.kernels()
    return K.ffn_forward(*K.aligned_rows(x, wg, wu, wd), "silu", keep=True)[1]


SIZES = [(1, 72, 33), (5, 256, 136), (128, 72, 200), (128, 256, 1000), (129, 72, 33), (300, 256, 200), (700, 136, 1000)]


@pytest.mark.parametrize("T,hid,inn", SIZES)
@pytest.mark.parametrize("dtype", [BF, F16])
def test_the_planes_hold_24_bits(T, hid, inn, dtype):
    x, wg, wu, wd, _ = make(T, hid, inn, dtype, seed=T)
    got = kept_values(keep(x, wg, wu, wd), T, inn)
    for name, g, w in zip("au", got, (wg, wu)):
        x64, w64 = x.double(), w.double()
        want = x64 @ w64.T
        reduction = hid * orc.U * (x64.abs() @ w64.abs().T)
        bound = reduction + 2.0**-16 * (want.abs() + reduction)
        over = (g.double() - want).abs() - bound
        assert over.max() <= 0, f"{name}: {float(over.max()):.3e} more than allowed"


@pytest.mark.parametrize("T,hid,inn", SIZES)
def test_whole_numbers_come_back_as_they_are(T, hid, inn):
    gen = torch.Generator(device="cuda").manual_seed(T)
    whole = lambda *s: torch.randint(-8, 8, s, generator=gen, device="cuda").to(BF)      # noqa: E731
    x, wg, wu, wd = whole(T, hid), whole(inn, hid), whole(inn, hid), whole(8, inn)      # sums below 64 * 256 = 2^14
    a, u = kept_values(keep(x, wg, wu, wd), T, inn)
    assert torch.equal(a.double(), x.double() @ wg.double().T) and torch.equal(u.double(), x.double() @ wu.double().T)


@pytest.mark.parametrize("T,hid,inn", [(128, 512, 1024), (300, 256, 384), (1000, 512, 1024)])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_two_roundings_behind_every_result(T, hid, inn, act, dtype):
    ins = make(T, hid, inn, dtype, seed=inn)
    want = orc.evaluate(*ins[:4], act, ins[4])
    leaves = [t.clone().requires_grad_() for t in ins[:4]]
    y = gdn2.gated_feed_forward(*leaves, act)
    half = torch.finfo(dtype).eps / 2
    for name, got in zip(("y", *NAMES), (y.detach(), *torch.autograd.grad(y, leaves, ins[4]))):
        value = want[name][0]
        rel = float((got.double() - value).norm() / value.norm())
        assert rel <= (2 / 3)**0.5 * half, f"{name}: {rel / half:.3f} half steps of the 2-norm"
