"""A captured decode step of a gated recurrent block, replayed over the tokens of a prompt: the eager steps' bits."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("B,D", [(1, 128), (5, 128), (3, 33)])
@pytest.mark.parametrize("n", [1, 4])
def test_a_captured_recurrence_step(B, D, n):
    gen = torch.Generator(device="cuda").manual_seed(D)
    v = torch.randn(B, 12, D, generator=gen, device="cuda").to(BF)
    g = -torch.rand(B, 12, D, generator=gen, device="cuda")
    w = torch.rand(B, 12, D, generator=gen, device="cuda").to(BF)
    state = torch.randn(B, D, generator=gen, device="cuda")
    eager = state.clone()
    want = [gdn2.gated_recurrence_decode(v[:, t:t + n], g[:, t:t + n], w[:, t:t + n], eager) for t in range(0, 12, n)]
    rows = [t[:, :n].clone() for t in (v, g, w)]
    held = state.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = gdn2.gated_recurrence_decode(*rows, held)
    held.copy_(state)                                  # a capture runs nothing
    for i, t in enumerate(range(0, 12, n)):
        for row, x in zip(rows, (v, g, w)):
            row.copy_(x[:, t:t + n])
        graph.replay()
        assert torch.equal(o, want[i])
    assert torch.equal(held, eager)


def test_two_captured_steps_of_one_block():
    """Token mixer and channel mixer in one graph, two graphs of two conversations replayed in turn: nothing is shared."""
    torch.manual_seed(0)
    mlp = gdn2.GatedFeedForward(128, 320).cuda().to(BF)
    proj = (torch.randn(3 * 128, 128, device="cuda") * 0.1).to(BF)

    @torch.no_grad()
    def step(x, state):
        v, w, g = (x @ proj.t()).split(128, -1)
        x = x + gdn2.gated_recurrence_step(v, -torch.nn.functional.softplus(g.float()), torch.sigmoid(w), state)
        return x + mlp(x)

    tokens = [torch.randn(9, B, 128, device="cuda").to(BF) for B in (1, 6)]
    want, eager = [], [torch.zeros(B, 128, device="cuda") for B in (1, 6)]
    for i in range(9):
        want.append([step(t[i], s) for t, s in zip(tokens, eager)])
    held, slots, outs, graphs = [torch.zeros(B, 128, device="cuda") for B in (1, 6)], [t[0].clone() for t in tokens], [], []
    for x, s in zip(slots, held):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(x, s))
    for i in range(9):
        for x, t in zip(slots, tokens):
            x.copy_(t[i])
        for graph in graphs:
            graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))
    assert all(torch.equal(a, b) for a, b in zip(held, eager))
