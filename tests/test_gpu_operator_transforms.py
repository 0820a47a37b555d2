"""Forward-mode tangents and tracers on the device: the calls that go through the host extension refuse them, too, forward and backward."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import gdn2_tilelang_b200 as gdn2
from gdn2_tilelang_b200 import _cabi

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _recurrence():
    g = -torch.rand(2, 70, 24, device="cuda")
    return gdn2.gated_recurrence, [torch.randn_like(g), g, torch.rand_like(g), torch.randn(2, 24, device="cuda")]


def _feed_forward():
    n = lambda *s: (torch.randn(*s, device="cuda") * 0.1).to(BF)              # noqa: E731
    return gdn2.gated_feed_forward, [n(7, 64), n(40, 64), n(40, 64), n(64, 40)]


MAKE = {"recurrence": _recurrence, "feed_forward": _feed_forward}


@pytest.fixture(params=["extension", "python"], autouse=True)
def way(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_cabi.kernels(), "host", None)


@pytest.mark.parametrize("name", MAKE)
@pytest.mark.parametrize("other_requires_grad", [False, True])
def test_an_input_with_a_tangent(name, other_requires_grad):
    call, ins = MAKE[name]()
    if other_requires_grad:
        ins[0].requires_grad_()
    for which in range(4):
        with forward_ad.dual_level():
            dual = list(ins)
            dual[which] = forward_ad.make_dual(ins[which], torch.ones_like(ins[which]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(*dual)
    with forward_ad.dual_level():                                            # a level without tangents is a plain call
        out = call(*ins)
    assert torch.isfinite(out[0] if isinstance(out, tuple) else out).all()


@pytest.mark.parametrize("name", MAKE)
def test_a_gradient_with_a_tangent(name):
    call, ins = MAKE[name]()
    ins[0].requires_grad_()
    out = call(*ins)
    out = out[0] if isinstance(out, tuple) else out
    with forward_ad.dual_level():
        dy = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, ins[0], dy)


def test_a_decoded_token_with_a_tangent():
    g = -torch.rand(2, 1, 24, device="cuda")
    state = torch.zeros(2, 24, device="cuda")
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        gdn2.gated_recurrence_decode(forward_ad.make_dual(g, torch.ones_like(g)), g, None, state)
    assert not state.any()


@pytest.mark.parametrize("name", MAKE)
def test_a_trace(name):
    from torch.fx.experimental.proxy_tensor import make_fx

    call, ins = MAKE[name]()
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(lambda x: call(x, *ins[1:]))(ins[0])
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(lambda x: call(x, *ins[1:]), (ins[0],))
    leaf = ins[0].clone().requires_grad_()
    out = call(leaf, *ins[1:])
    out = out[0] if isinstance(out, tuple) else out
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(lambda dy: torch.autograd.grad(out, leaf, dy, retain_graph=True)[0])(torch.ones_like(out))
    assert torch.isfinite(torch.autograd.grad(out, leaf, torch.ones_like(out))[0]).all()


@pytest.mark.parametrize("name", MAKE)
def test_a_mode_that_counts(name):
    from torch.utils.flop_counter import FlopCounterMode

    call, ins = MAKE[name]()
    first = lambda out: out[0] if isinstance(out, tuple) else out             # noqa: E731
    want = first(call(*ins))
    with FlopCounterMode(display=False):
        got = first(call(*ins))
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", MAKE)
@pytest.mark.parametrize("way", ["extension"], indirect=True)
def test_a_compiled_caller(name, way):
    """A compiler that captures what it can runs the extension's call as it is, between its captured parts."""
    call, ins = MAKE[name]()
    first = lambda out: out[0] if isinstance(out, tuple) else out             # noqa: E731

    def block(*a):
        return first(call(*(t * 1 for t in a))) + 1

    leaves = [t.clone().requires_grad_() for t in ins]
    want = block(*leaves)
    dy = torch.ones_like(want)
    grads = torch.autograd.grad(want, leaves, dy)
    torch._dynamo.reset()
    got = torch.compile(block, backend="eager")(*leaves)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, dy), grads))
