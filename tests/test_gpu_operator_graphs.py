"""The gated operators inside autograd's own machinery: activation checkpoints, hooks on saved tensors, inputs without tokens."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu


def _recurrence(packed=False, size=(2, 70, 24)):
    from gdn2_tilelang_b200 import gated_recurrence

    torch.manual_seed(1)
    B, S, D = (1, *size[1:]) if packed else size
    cu = [0, 30, 30, S] if packed else None
    v, w = (torch.randn(B, S, D, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    g = (-torch.rand(B, S, D, device="cuda")).requires_grad_()
    state = torch.randn(3 if packed else B, D, device="cuda").requires_grad_()

    def call(v, g, w, state):
        o, final = gated_recurrence(v, g, w, state, output_final_state=True, cu_seqlens=cu)
        return torch.cat((o.float().flatten(), final.flatten()))

    return call, (v, g, w, state)


def _feed_forward(tokens=7):
    from gdn2_tilelang_b200 import gated_feed_forward

    torch.manual_seed(2)
    x = torch.randn(tokens, 72, device="cuda").bfloat16()
    weights = [(torch.randn(*s, device="cuda") * 0.1).bfloat16() for s in ((40, 72), (40, 72), (72, 40))]
    return gated_feed_forward, tuple(t.requires_grad_() for t in (x, *weights))


CASES = {"recurrence": lambda: _recurrence(), "packed": lambda: _recurrence(True), "feed_forward": lambda: _feed_forward(),
         "feed_forward_many": lambda: _feed_forward(200)}


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("early_stop", [True, False])
def test_under_a_checkpoint(case, reentrant, early_stop):
    """The same bits as without one: the kernels' order of summation depends on the sizes alone."""
    from torch.utils.checkpoint import set_checkpoint_early_stop

    call, ins = CASES[case]()
    dy = torch.randn_like(call(*ins))
    want = torch.autograd.grad(call(*ins), ins, dy)
    with set_checkpoint_early_stop(early_stop):
        y = checkpoint(call, *ins, use_reentrant=reentrant)
        y.backward(dy)
    for t, x in zip(ins, want):
        assert torch.equal(t.grad, x)


class _Stop(Exception):
    pass


@pytest.mark.parametrize("case", CASES)
def test_an_exception_of_a_hook_keeps_its_type(case):
    call, ins = CASES[case]()

    def pack(t):
        raise _Stop("stop")

    with pytest.raises(_Stop), torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        call(*ins)
    assert all(torch.isfinite(x).all() for x in torch.autograd.grad(call(*ins).sum(), ins))     # and the next call is whole


@pytest.mark.parametrize("shape", [(2, 0, 24), (0, 5, 24), (2, 5, 0)])
@pytest.mark.parametrize("with_state", [False, True])
def test_gradients_without_tokens(shape, with_state):
    from gdn2_tilelang_b200 import gated_recurrence

    v, w = (torch.randn(shape, device="cuda").half().requires_grad_() for _ in range(2))
    g = torch.zeros(shape, device="cuda").requires_grad_()
    state = torch.randn(shape[0], shape[2], device="cuda").requires_grad_() if with_state else None
    o, final = gated_recurrence(v, g, w, state, output_final_state=True)
    assert o.dtype == torch.float16 and o.shape == shape and final.shape == (shape[0], shape[2])
    (o.float().sum() + final.sum()).backward()
    assert v.grad.shape == g.grad.shape == w.grad.shape == shape
    if with_state:
        assert torch.equal(state.grad, torch.ones_like(state))
