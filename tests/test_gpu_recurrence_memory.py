"""Slow decays: what is left of a one-sided error of the decay after thousands of tokens.

With a memory of N tokens a decay that is off by e one way puts the state off by e N / sqrt(2) in the 2-norm (sum of k^2 a^2k against
sum of a^2k). Roundings to nearest go both ways: three a token (the decay, a product and a sum, or their composition), at most
u / sqrt(3) of the value each in the mean square, which leaves u sqrt(N / 2), u = 2^-24. For N = 2000 that is 1.9e-6, and a
tenth of a unit one way 8.4e-6: 3e-6 tells them apart. At |g| = 1/32, where the kernel changes its formula, N is 32: below it
2.4e-7 and the polynomial's remainder, 3e-10 N; above it the approximate instruction may be off by 4 units one way, 5.4e-6."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2

pytestmark = pytest.mark.gpu
U = 2.0**-24
GROUPS = {"slow": (slice(0, 64), 3e-6), "below": (slice(64, 128), 1.5 * (U * 4 + 3e-10 * 32)), "above": (slice(128, 192), U * 4 + 4 * U * 32 / 2**0.5)}


def make(S, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.randn(4, S, 192, generator=gen, device="cuda")
    r = torch.rand(4, S, 192, generator=gen, device="cuda")
    g = torch.empty_like(v)
    g[..., :64] = -1e-3 * r[..., :64]
    edge = torch.tensor(1 / 32, device="cuda")
    g[..., 64:128] = -(edge * (1 - 2.0**-10 * r[..., 64:128] - 2.0**-20))
    g[..., 128:] = -(edge * (1 + 2.0**-10 * r[..., 128:]))
    assert (g[..., 64:128].abs() < 1 / 32).all() and (g[..., 128:].abs() >= 1 / 32).all()
    return v, g


def last_state(v, g):
    G = g.double().cumsum(1)
    return ((G[:, -1:] - G).exp() * v.double()).sum(1)


@pytest.mark.parametrize("S", [32768, 20001])
def test_the_state_after_many_tokens(S):
    v, g = make(S, S)
    fin = gdn2.gated_recurrence(v, g, output_final_state=True)[1]
    want = last_state(v, g)
    for name, (at, bound) in GROUPS.items():
        rel = float((fin[..., at].double() - want[..., at]).norm() / want[..., at].norm())
        assert rel <= bound, f"{name}: {rel:.2e} of the 2-norm"


def test_the_same_token_by_token():
    """In place, 8 tokens a call."""
    v, g = make(16384, 7)
    state = torch.zeros(4, 192, device="cuda")
    for t in range(0, v.shape[1], 8):
        gdn2.gated_recurrence_decode(v[:, t:t + 8], g[:, t:t + 8], None, state)
    want = last_state(v, g)
    for name, (at, bound) in GROUPS.items():
        rel = float((state[..., at].double() - want[..., at]).norm() / want[..., at].norm())
        assert rel <= bound, f"{name}: {rel:.2e} of the 2-norm"


def test_the_gradient_of_the_initial_state_after_many_tokens():
    """c_0 = sum of exp(g_1 + .. + g_t) do_t: the same sums from the other end."""
    v, g = make(20001, 3)
    state = torch.zeros(4, 192, device="cuda", requires_grad=True)
    o, _ = gdn2.gated_recurrence(v, g, None, state)
    got = torch.autograd.grad(o, state, v)[0]
    want = (g.double().cumsum(1).exp() * v.double()).sum(1)
    for name, (at, bound) in GROUPS.items():
        rel = float((got[..., at].double() - want[..., at]).norm() / want[..., at].norm())
        assert rel <= bound, f"{name}: {rel:.2e} of the 2-norm"
