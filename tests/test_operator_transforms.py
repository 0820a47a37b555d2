"""The gated operators under autograd's forward mode and under tracers: their kernels run where a transform cannot see them, so what
it would get silently wrong is refused. No GPU."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import gdn2_tilelang_b200 as gdn2
from gdn2_tilelang_b200 import _cabi

BF = torch.bfloat16


@pytest.fixture(autouse=True)
def any_device(monkeypatch):
    """Host tensors pass the device check; no kernel may be reached."""
    monkeypatch.setattr(_cabi, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(_cabi, "kernels", lambda: pytest.fail("a refused call reached the kernels"))


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


CALLS = {
    "recurrence": (lambda v, g, w, s: gdn2.gated_recurrence(v, g, w, s), lambda: [z(2, 4, 8) for _ in range(3)] + [z(2, 8)]),
    "packed": (lambda v, g, w, s: gdn2.gated_recurrence(v, g, w, s, cu_seqlens=[0, 1, 4]), lambda: [z(1, 4, 8) for _ in range(3)] + [z(2, 8)]),
    "no_tokens": (lambda v, g, w, s: gdn2.gated_recurrence(v, g, w, s), lambda: [z(2, 0, 8) for _ in range(3)] + [z(2, 8)]),
    "decode": (gdn2.gated_recurrence_decode, lambda: [z(2, 3, 8) for _ in range(3)] + [z(2, 8)]),
    "step": (gdn2.gated_recurrence_step, lambda: [z(2, 8) for _ in range(4)]),
    "feed_forward": (gdn2.gated_feed_forward, lambda: [z(3, 8, dtype=BF), z(16, 8, dtype=BF), z(16, 8, dtype=BF), z(8, 16, dtype=BF)]),
    "feed_forward_no_tokens": (gdn2.gated_feed_forward,
                               lambda: [z(0, 8, dtype=BF), z(16, 8, dtype=BF), z(16, 8, dtype=BF), z(8, 16, dtype=BF)]),
}


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("name", CALLS)
def test_a_tangent_is_refused(name, which):
    call, make = CALLS[name]
    ins = make()
    with forward_ad.dual_level():
        ins[which] = forward_ad.make_dual(ins[which], torch.ones_like(ins[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(*ins)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):      # which does not end forward mode
            call(*ins)


@pytest.mark.parametrize("name", ["recurrence", "feed_forward"])
def test_a_jacobian_vector_product_is_refused(name):
    call, make = CALLS[name]
    ins = make()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda x: call(x, *ins[1:]), (ins[0],), (torch.ones_like(ins[0]),))


def test_a_decay_of_another_type_keeps_its_tangent():
    v, g = z(2, 4, 8), z(2, 4, 8, dtype=BF)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        gdn2.gated_recurrence(v, forward_ad.make_dual(g, torch.ones_like(g)))


class _Call(torch.nn.Module):
    def __init__(self, call, ins):
        super().__init__()
        self.call, self.rest = call, ins[1:]

    def forward(self, x):
        out = self.call(x, *self.rest)
        return out[0] if isinstance(out, tuple) else out


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
@pytest.mark.parametrize("pre_dispatch", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_a_trace_is_refused(name, mode, pre_dispatch):
    """The recorded graph would hold an empty tensor in the place of the result."""
    from torch.fx.experimental.proxy_tensor import make_fx

    call, make = CALLS[name]
    ins = make()
    if mode == "real":
        fn, args = _Call(call, ins), (ins[0],)
    else:
        fn, args = (lambda *a: call(*a)), tuple(ins)
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(fn, tracing_mode=mode, pre_dispatch=pre_dispatch)(*args)


@pytest.mark.parametrize("name", CALLS)
def test_a_scripted_trace_is_refused(name):
    call, make = CALLS[name]
    ins = make()
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(_Call(call, ins), (ins[0],))


def test_fake_results_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode

    v = z(2, 4, 8)
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(NotImplementedError, match="traced"):
        gdn2.gated_recurrence(v, v)


def test_other_modes_are_not(monkeypatch):
    """A mode that records nothing (counting, logging) does not refuse the call: it gets as far as the kernels."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Passing(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    class Reached(Exception):
        pass

    def reached():
        raise Reached

    monkeypatch.setattr(_cabi, "kernels", reached)
    for name, (call, make) in CALLS.items():
        if "no_tokens" not in name:
            with Passing(), pytest.raises(Reached):
                call(*make())
