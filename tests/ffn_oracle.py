"""The gated feed-forward block and its gradient in 64 bits, with bounds on what a 16-bit evaluation may be off by.

Elementwise bounds: a product of K terms summed in float32 is off by at most K 2^-24 of the sum of the terms' magnitudes, the
activation's approximate instructions by 2^-19 of it, every rounding to 16 bits by half a step, and all of it is carried on
through the next products term by term (|act'| < 1.13, |act''| < 0.8). Such a bound grows with the sum of magnitudes while the
result grows with its root, so long reductions get a second one: roundings are independent of one another, so in the
2-norm each adds at most half a step of what it rounds. Forward there are two in a row (h, y); in a gradient up to four (a or u, da
or du, h, the result), the second of them through a factor that varies as a and u do, which is given 1.5."""

from __future__ import annotations

import math

import torch

U = 2.0**-24


def activation(a, name):
    """``act(a), act'(a)``."""
    if name == "silu":
        s = torch.sigmoid(a)
        return a * s, s + a * s * (1 - s)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (a + 0.044715 * a**3))
    return 0.5 * a * (1 + t), 0.5 * (1 + t) + 0.5 * a * (1 - t * t) * c * (1 + 3 * 0.044715 * a * a)


def evaluate(x, wg, wu, wd, act_name, dy=None):
    """``{name: (value, bound)}`` for y and, with ``dy``, dx, dw_gate, dw_up, dw_down."""
    half = torch.finfo(x.dtype).eps / 2
    x, wg, wu, wd = (t.detach().double() for t in (x, wg, wu, wd))
    hid, inn, T = x.shape[1], wg.shape[0], x.shape[0]
    dot = lambda p, q, k: k * U * (p.abs() @ q.abs())             # noqa: E731
    a, u = x @ wg.T, x @ wu.T
    ea, eu = dot(x, wg.T, hid), dot(x, wu.T, hid)
    act, slope = activation(a, act_name)
    h = act * u
    eh = 1.13 * ea * (u.abs() + eu) + act.abs() * eu + 2.0**-18 * h.abs()
    eh = eh + half * (h.abs() + eh) + 1e-7                        # (1e-7: under fp16's smallest normal number)
    y = h @ wd.T
    out = {"y": (y, eh @ wd.abs().T + dot(h.abs() + eh, wd.T, inn))}
    if dy is None:
        return out
    dy = dy.detach().double()
    ea, eu = ea + half * (a.abs() + ea) + 1e-7, eu + half * (u.abs() + eu) + 1e-7      # as they are kept
    dh, edh = dy @ wd, dot(dy, wd, wd.shape[0])
    da, du = dh * u * slope, dh * act
    eda = edh * (u.abs() + eu) * 1.13 + dh.abs() * (1.13 * eu + 0.8 * ea * (u.abs() + eu)) + 2.0**-17 * (dh * u).abs()
    edu = edh * (act.abs() + 1.13 * ea) + dh.abs() * 1.13 * ea + 2.0**-18 * du.abs()
    eda, edu = eda + half * (da.abs() + eda) + 1e-7, edu + half * (du.abs() + edu) + 1e-7
    out["dx"] = (da @ wg + du @ wu, eda @ wg.abs() + edu @ wu.abs() + 2 * inn * U * ((da.abs() + eda) @ wg.abs() + (du.abs() + edu) @ wu.abs()))
    out["dw_gate"] = (da.T @ x, eda.T @ x.abs() + dot((da.abs() + eda).T, x, T))
    out["dw_up"] = (du.T @ x, edu.T @ x.abs() + dot((du.abs() + edu).T, x, T))
    out["dw_down"] = (dy.T @ h, dy.abs().T @ eh + dot(dy.T, h.abs() + eh, T))
    return out


def assert_within(got, want, bound, what):
    info = torch.finfo(got.dtype)
    half = info.eps / 2
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}"
    got = got.detach().double().to(want.device)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - want).abs()
    over = off - (bound + half * (want.abs() + bound) + info.smallest_normal)
    assert over.max() <= 0, f"{what}: off by {float(off.flatten()[over.argmax()]):.3e}, {float(over.max()):.3e} more than allowed"
    if got.numel() >= 256:
        roundings = 2 if what == "y" else 5.5
        rel = float((got - want).norm() / want.norm())
        assert rel <= roundings * half, f"{what}: {rel:.3e} of the 2-norm"
