"""Every buffer the recurrence writes between guard rows of a larger one: odd channel counts, partial tiles, packed ends."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from gdn2_tilelang_b200 import _cabi
from tests import recurrence_oracle as orc
from tests.test_gpu_recurrence import BF, F16, F32, check_forward, make, on_gpu

pytestmark = pytest.mark.gpu
GUARD = 512


@pytest.fixture
def guarded(monkeypatch):
    """What ``torch.empty`` and ``torch.empty_like`` make lies between guards, and calls go through Python, which makes its
    buffers with them. Calling the fixture checks the guards of all of them."""
    K = _cabi.kernels()
    monkeypatch.setattr(K, "host", None)
    real, made = torch.empty, []

    def empty(*shape, dtype=None, device=None):
        shape = tuple(shape[0]) if len(shape) == 1 and not isinstance(shape[0], int) else shape
        n = 1
        for s in shape:
            n *= s
        buf = real(n + 2 * GUARD, dtype=dtype, device=device).fill_(7.0)
        made.append((buf, n))
        return buf[GUARD:GUARD + n].view(shape)

    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(torch, "empty_like", lambda t: empty(*t.shape, dtype=t.dtype, device=t.device))

    def verify(at_least):
        monkeypatch.setattr(torch, "empty", real)
        torch.cuda.synchronize()
        assert len(made) >= at_least
        for buf, n in made:
            assert (buf[:GUARD] == 7).all() and (buf[GUARD + n:] == 7).all()
        K.check_device_status()

    return verify


@pytest.mark.parametrize("D", [33, 72, 1001])
@pytest.mark.parametrize("B,S", [(2, 1), (3, 61), (1, 130), (2, 1001)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_forward_and_backward(B, S, D, dtype, guarded):
    v, g, w, s = make(B, S, D, dtype, seed=S)
    gen = torch.Generator().manual_seed(9)
    do, df = torch.randn(B, S, D, generator=gen).to(dtype), torch.randn(B, D, generator=gen)
    ins = on_gpu(v, g, w, s, grad=True)
    o, fin = gdn2.gated_recurrence(*ins, output_final_state=True)
    grads = torch.autograd.grad((o, fin), ins, (do.cuda(), df.cuda()))
    guarded(7)                                         # o, final, marks, dv, dg, dw, dstate
    check_forward(o, fin, orc.scan(v, g, w, s))
    want, bound = orc.gradients(v, g, w, s, do, df)
    for name, y, x, e in zip("vgws", grads, want, bound):
        orc.assert_within(y, x, e, f"d{name}")


@pytest.mark.parametrize("D,dtype", [(33, BF), (72, F16), (1001, F32)])
@pytest.mark.parametrize("cu", [[0, 1, 1, 66], [0, 0, 129, 200, 200], [0, 300]], ids=str)
def test_packed(cu, D, dtype, guarded):
    N = len(cu) - 1
    v, g, w, s = make(1, cu[-1], D, dtype, sequences=N, seed=N)
    do, df = torch.ones(v.shape).to(dtype), torch.ones(N, D)
    ins = on_gpu(v, g, w, s, grad=True)
    o, fin = gdn2.gated_recurrence(*ins, output_final_state=True, cu_seqlens=cu)
    grads = torch.autograd.grad((o, fin), ins, (do.cuda(), df.cuda()))
    guarded(7)
    check_forward(o, fin, orc.scan(v, g, w, s, cu))
    want, bound = orc.gradients(v, g, w, s, do, df, cu)
    for name, y, x, e in zip("vgws", grads, want, bound):
        orc.assert_within(y, x, e, f"d{name}")


@pytest.mark.parametrize("D,dtype", [(33, BF), (72, F16), (1001, F32)])
@pytest.mark.parametrize("n", [1, 3, 8, 30])
def test_decode(n, D, dtype, guarded):
    v, g, w, s = make(3, n, D, dtype, seed=n)
    vc, gc, wc = on_gpu(v, g, w)
    state = torch.empty(3, D, dtype=F32, device="cuda").copy_(s)      # between guards, too, and updated in place
    o = gdn2.gated_recurrence_decode(vc, gc, wc, state)
    guarded(2)
    check_forward(o, state, orc.scan(v, g, w, s))
