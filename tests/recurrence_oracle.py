"""The diagonal recurrence and its gradient in 64 bits, with a bound on what a float32 evaluation of it may be off by.

The bound: a step multiplies by a decay that is off by at most 4 units u = 2^-24 of its value (the approximate exponential's
2^-22; one unit where a polynomial takes its place), and by |g| units more, because the exponential's argument g log2(e) is
rounded (u of it, and exp turns an absolute error into a relative one). It rounds a product and a sum; composing runs of
tokens rounds two more. 8 u of the magnitude that passes a step covers these, and what has accumulated is carried on by the same
decays: with the magnitudes m_t = a_t m_{t-1} + |x_t|, the bound is e_t = a_t (e_{t-1} + |g_t| u m_{t-1}) + 8 u m_t. (Where
exp(g) underflows both terms of the product with |g| are 0.)"""

from __future__ import annotations

import torch

U = 2.0**-24
STEP = 8 * U


def rounded(g):
    """The error of the rounded argument of exp(g), relative."""
    return U * g.abs().clamp(max=1e3)


def scan(v, g, w, state, bounds=None):
    """``[B, S, D]`` inputs of any type; returns float64 ``o, final, err_o, err_final`` (``bounds``: offsets of packed sequences)."""
    v, g = v.detach().double(), g.detach().double()
    x = v if w is None else v * w.detach().double()
    B, S, D = v.shape
    seqs = [(slice(b, b + 1), 0, S) for b in range(B)] if bounds is None else [(slice(0, 1), lo, hi) for lo, hi in zip(bounds, bounds[1:])]
    o, err = torch.zeros_like(v), torch.zeros_like(v)
    fin, efin = v.new_zeros(len(seqs), D), v.new_zeros(len(seqs), D)
    for i, (b, lo, hi) in enumerate(seqs):
        h = v.new_zeros(1, D) if state is None else state[i:i + 1].detach().double()
        m, e = h.abs(), torch.zeros_like(h)
        for t in range(lo, hi):
            a = g[b, t].exp()
            e, m = a * (e + rounded(g[b, t]) * m), a * m + x[b, t].abs()
            h, e = a * h + x[b, t], e + STEP * m
            o[b, t], err[b, t] = h, e
        fin[i], efin[i] = h, e
    return o, fin, err, efin


def gradients(v, g, w, state, do, dfinal, bounds=None):
    """float64 ``(dv, dg, dw, dstate)`` and their bounds; ``dw`` is that of a gate of ones where ``w`` is ``None``."""
    o, _, err, _ = scan(v, g, w, state, bounds)
    v, g = v.detach().double(), g.detach().double()
    wd = torch.ones_like(v) if w is None else w.detach().double()
    B, S, D = v.shape
    seqs = [(slice(b, b + 1), 0, S) for b in range(B)] if bounds is None else [(slice(0, 1), lo, hi) for lo, hi in zip(bounds, bounds[1:])]
    dv, dg, dw = torch.zeros_like(v), torch.zeros_like(v), torch.zeros_like(v)
    ev, eg, ew = torch.zeros_like(v), torch.zeros_like(v), torch.zeros_like(v)
    ds, es = v.new_zeros(len(seqs), D), v.new_zeros(len(seqs), D)
    do = torch.zeros_like(v) if do is None else do.detach().double()
    for i, (b, lo, hi) in enumerate(seqs):
        c = v.new_zeros(1, D) if dfinal is None else dfinal[i:i + 1].detach().double()
        m, e = c.abs(), torch.zeros_like(c)
        h0 = v.new_zeros(1, D) if state is None else state[i:i + 1].detach().double()
        for t in range(hi - 1, lo - 1, -1):
            a = g[b, t].exp()
            dh, mh = do[b, t] + c, do[b, t].abs() + m
            before, eb = (o[b, t - 1], err[b, t - 1]) if t > lo else (h0, torch.zeros_like(h0))
            eh = e + 2 * U * mh                       # the sum do + c
            dv[b, t], ev[b, t] = dh * wd[b, t], (eh + U * dh.abs()) * wd[b, t].abs()
            dw[b, t], ew[b, t] = dh * v[b, t], (eh + U * dh.abs()) * v[b, t].abs()
            c, m, e = a * dh, a * mh, a * (e + rounded(g[b, t]) * mh) + STEP * a * mh
            dg[b, t] = c * before
            eg[b, t] = (c.abs() + e) * (eb + STEP * before.abs()) + before.abs() * e
        ds[i], es[i] = c, e
    return (dv, dg, dw, ds), (ev, eg, ew, es)


def assert_within(got, want, bound, what):
    """``got`` within ``bound`` of ``want`` plus half a step of its own type."""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal
    off = (got.detach().double().cpu() - want).abs()
    over = off - (bound + half * (want.abs() + bound) + tiny)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert over.max() <= 0, f"{what}: off by {float(off.flatten()[over.argmax()]):.3e}, {float(over.max()):.3e} more than allowed"
