"""The gated operators as programs around them use them: results written in place, calls from several threads, inputs changed before the
backward pass, the backward pass twice."""

from __future__ import annotations

import threading

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from gdn2_tilelang_b200 import _cabi
from tests.test_gpu_feed_forward import make as make_ffn
from tests.test_gpu_recurrence import BF, make, on_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "python"], autouse=True)
def way(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_cabi.kernels(), "host", None)


def _recurrence(shape4=False):
    ins = on_gpu(*make(2, 130, 48, BF))
    if shape4:
        ins = [t.view(*t.shape[:-1], 6, 8) for t in ins]
    return (lambda *a: gdn2.gated_recurrence(*a, output_final_state=True)), [t.requires_grad_() for t in ins]


def _feed_forward():
    x, wg, wu, wd, _ = make_ffn(130, 72, 136, BF)
    return (lambda *a: (gdn2.gated_feed_forward(*a),)), [t.requires_grad_() for t in (x, wg, wu, wd)]


CASES = {"recurrence": _recurrence, "recurrence_heads": lambda: _recurrence(True), "feed_forward": _feed_forward}


@pytest.mark.parametrize("case", CASES)
def test_results_written_in_place(case):
    """A residual added into the result: the gradients are those of the sum."""
    call, ins = CASES[case]()
    want = torch.autograd.grad([o.float().square().sum() for o in call(*ins)], ins)
    outs = call(*ins)
    add = [torch.randn_like(o) for o in outs]
    wanted = torch.autograd.grad([((o + a).float().square()).sum() for o, a in zip(call(*ins), add)], ins)
    for o, a in zip(outs, add):
        o += a
    got = torch.autograd.grad([o.float().square().sum() for o in outs], ins)
    assert all(torch.equal(a, b) for a, b in zip(got, wanted)) and not torch.equal(got[0], want[0])


@pytest.mark.parametrize("case", CASES)
def test_an_input_changed_before_the_backward_pass(case):
    call, ins = CASES[case]()
    for which in (0, 1):
        outs = call(*ins)
        with torch.no_grad():
            ins[which].mul_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            outs[0].float().sum().backward()


@pytest.mark.parametrize("case", CASES)
def test_the_backward_pass_twice(case):
    call, ins = CASES[case]()
    o = call(*ins)[0]
    dy = torch.randn_like(o)
    first = torch.autograd.grad(o, ins, dy, retain_graph=True, allow_unused=True)
    second = torch.autograd.grad(o, ins, dy, allow_unused=True)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(o, ins, dy)


def test_several_threads_at_once():
    """Eight threads, each on a stream of its own, forward and backward: the bits of one thread alone."""
    work = []
    for i, case in enumerate(["recurrence", "feed_forward"] * 4):
        call, ins = CASES[case]()
        ins = [t.detach().clone().requires_grad_() for t in ins]
        o = call(*ins)[0]
        dy = torch.randn_like(o)
        work.append((call, ins, dy, o.detach(), torch.autograd.grad(o, ins, dy)))
    torch.cuda.synchronize()
    failed = []

    def run(call, ins, dy, want, grads):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(30):
                    o = call(*ins)[0]
                    got = torch.autograd.grad(o, ins, dy)
                    ok = torch.equal(o, want) and all(torch.equal(a, b) for a, b in zip(got, grads))
                    assert ok
        except BaseException as e:      # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
