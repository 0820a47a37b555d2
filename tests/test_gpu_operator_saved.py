"""Tensors that the gated operators save, brought back by a program's hooks: from the host, in another layout, as something else."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from gdn2_tilelang_b200 import _cabi
from tests.test_gpu_feed_forward import make as make_ffn
from tests.test_gpu_recurrence import BF, F32, make, on_gpu

pytestmark = pytest.mark.gpu
hooks = torch.autograd.graph.saved_tensors_hooks


@pytest.fixture(params=["extension", "python"], autouse=True)
def way(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_cabi.kernels(), "host", None)


def _recurrence(D, dtype, packed=False):
    cu = [0, 70, 70, 130] if packed else None
    ins = on_gpu(*make(1 if packed else 2, 130, D, dtype, sequences=3 if packed else None), grad=True)
    return (lambda *a: gdn2.gated_recurrence(*a, output_final_state=True, cu_seqlens=cu)), ins


def _feed_forward(T, hid, inn, out):
    x, wg, wu, wd, _ = make_ffn(T, hid, inn, BF, out)
    return (lambda *a: (gdn2.gated_feed_forward(*a),)), [t.requires_grad_() for t in (x, wg, wu, wd)]


CASES = {"recurrence": lambda: _recurrence(72, BF), "recurrence_odd": lambda: _recurrence(33, F32), "packed": lambda: _recurrence(72, BF, True),
         "feed_forward": lambda: _feed_forward(130, 72, 136, 72), "feed_forward_odd": lambda: _feed_forward(130, 71, 133, 69),
         "feed_forward_few_odd": lambda: _feed_forward(5, 71, 133, 69)}


def gradients(call, ins, pack=None, unpack=None):
    if pack is None:
        outs = call(*ins)
    else:
        with hooks(pack, unpack):
            outs = call(*ins)
    gen = torch.Generator(device="cuda").manual_seed(5)
    return torch.autograd.grad(outs, ins, [torch.randn(o.shape, generator=gen, device="cuda").to(o.dtype) for o in outs])


def apart(t):
    """The same values with every dimension's stride doubled and the last two swapped in memory."""
    if t.dim() < 2:
        return torch.stack([t, t], -1)[..., 0]
    return torch.stack([t.transpose(-1, -2)] * 2, -1)[..., 0].transpose(-1, -2)


@pytest.mark.parametrize("case", CASES)
def test_kept_on_the_host_meanwhile(case):
    call, ins = CASES[case]()
    want = gradients(call, ins)
    for got in (gradients(call, ins, lambda t: t.cpu(), lambda t: t.cuda()),
                gradients(call, ins, lambda t: t.to("cpu", memory_format=torch.contiguous_format), lambda t: t.cuda())):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.autograd.graph.save_on_cpu():
        outs = call(*ins)
    gen = torch.Generator(device="cuda").manual_seed(5)
    got = torch.autograd.grad(outs, ins, [torch.randn(o.shape, generator=gen, device="cuda").to(o.dtype) for o in outs])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("case", CASES)
def test_brought_back_in_another_layout(case):
    call, ins = CASES[case]()
    want = gradients(call, ins)
    got = gradients(call, ins, lambda t: t, apart)
    # rows are laid out again, so values may go through the kernels for unaligned rows: the same arithmetic, tile by tile of 64 tokens
    for a, b in zip(got, want):
        assert a.shape == b.shape and float((a.double() - b.double()).norm()) <= 2**-8 * float(b.double().norm())


CHANGES = {"type": lambda t: t.double() if t.is_floating_point() else t.int(), "shape": lambda t: t[:1] if t.shape[0] > 1 else t[..., :1],
           "device": lambda t: t.cpu(), "rank": lambda t: t.unsqueeze(0)}


@pytest.mark.parametrize("case", ["recurrence", "packed", "feed_forward"])
@pytest.mark.parametrize("change", CHANGES)
def test_brought_back_as_something_else(case, change):
    """One of the saved tensors after another; the checks stand before any launch."""
    call, ins = CASES[case]()
    seen = []
    gradients(call, ins, lambda t: seen.append(t) or t, lambda t: t)
    for which in range(len(seen)):
        count = []

        def pack(t):
            count.append(t)
            return len(count) - 1, t

        with pytest.raises((RuntimeError, ValueError)):
            gradients(call, ins, pack, lambda p: CHANGES[change](p[1]) if p[0] == which else p[1])
    assert all(torch.isfinite(t).all() for t in gradients(call, ins))
