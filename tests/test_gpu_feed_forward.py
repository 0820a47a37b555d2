"""``gated_feed_forward`` on the GPU against the same block in 64 bits (tolerances: tests/ffn_oracle.py)."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from tests import ffn_oracle as orc

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16
NAMES = ("dx", "dw_gate", "dw_up", "dw_down")


def make(T, hid, inn, dtype, out=None, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = out or hid
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")            # noqa: E731
    return n(T, hid).to(dtype), (n(inn, hid) * hid**-0.5).to(dtype), (n(inn, hid) * hid**-0.5).to(dtype), \
        (n(out, inn) * inn**-0.5).to(dtype), n(T, out).to(dtype)


def check(ins, act, grads=True):
    x, wg, wu, wd, dy = ins
    want = orc.evaluate(x, wg, wu, wd, act, dy if grads else None)
    with torch.no_grad():
        y = gdn2.gated_feed_forward(x, wg, wu, wd, act)
    orc.assert_within(y, *want["y"], "y")
    if grads:
        leaves = [t.detach().clone().requires_grad_() for t in (x, wg, wu, wd)]
        y2 = gdn2.gated_feed_forward(*leaves, act)
        assert torch.equal(y, y2)
        for name, g in zip(NAMES, torch.autograd.grad(y2, leaves, dy)):
            orc.assert_within(g, *want[name], name)


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 600, 1025])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_tokens(T, dtype):
    check(make(T, 256, 384, dtype, seed=T), "silu")


@pytest.mark.parametrize("T", [3, 40, 150, 700])
@pytest.mark.parametrize("hid,inn,out", [(8, 8, 8), (64, 64, 64), (72, 200, 40), (128, 136, 520), (1000, 88, 256), (264, 1032, 24),
                                         (1, 1, 1), (7, 100, 9), (100, 33, 100), (257, 131, 65), (513, 255, 1001)])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_sizes(T, hid, inn, out, act):
    check(make(T, hid, inn, BF, out, seed=hid), act)


@pytest.mark.parametrize("T,hid,inn", [(1, 2048, 5632), (24, 2048, 5632), (64, 1024, 4096), (65, 2048, 5632), (2100, 2048, 2816),
                                       (4096, 1024, 2816), (1003, 1001, 2731)])
def test_real_sizes(T, hid, inn):
    check(make(T, hid, inn, F16 if T == 24 else BF, seed=T), "silu", grads=T > 24)


def test_more_tiles_than_pairs_twice_over():
    """Both halves of tensor memory and every stage many times round."""
    check(make(3100, 520, 4100, BF), "gelu_tanh")


def test_leading_dimensions_and_strides():
    x, wg, wu, wd, _ = make(60, 96, 160, BF)
    want = gdn2.gated_feed_forward(x, wg, wu, wd)
    f = gdn2.gated_feed_forward
    assert torch.equal(f(x.view(3, 20, 96), wg, wu, wd), want.view(3, 20, 96))
    assert torch.equal(f(x[7], wg, wu, wd), f(x[7:8], wg, wu, wd)[0])
    wide = torch.full((60, 200), float("nan"), dtype=BF, device="cuda")
    for first in (8, 3):                                       # rows on 16 bytes, and not
        wide[:, first:first + 96] = x
        assert torch.equal(f(wide[:, first:first + 96], wg, wu, wd), want)
    both = torch.cat([wg, wu])                                 # halves of one weight
    assert torch.equal(f(x, both[:160], both[160:], wd), want)
    odd = torch.empty(160 * 96 + 1, dtype=BF, device="cuda")[1:].view(160, 96)
    odd.copy_(wg)
    assert torch.equal(f(x, odd, wu, wd), want)
    assert torch.equal(f(x, wg.t().contiguous().t(), wu, wd.t().contiguous().t()), want)
    one = x[:1].expand(60, -1)                                 # the same token over and over, not materialised
    assert torch.equal(f(one, wg, wu, wd), f(one.contiguous(), wg, wu, wd))


def test_no_tokens():
    x, wg, wu, wd, _ = make(4, 64, 64, BF)
    assert gdn2.gated_feed_forward(x[:0], wg, wu, wd).shape == (0, 64)
    leaves = [t.clone().requires_grad_() for t in (x[:0], wg, wu, wd)]
    y = gdn2.gated_feed_forward(leaves[0].view(2, 0, 64), *leaves[1:])
    grads = torch.autograd.grad(y.sum(), leaves)
    assert y.shape == (2, 0, 64) and all(g.shape == t.shape and not g.any() for g, t in zip(grads, leaves))


@pytest.mark.parametrize("T", [40, 300])
def test_gradients_of_some_inputs(T):
    x, wg, wu, wd, dy = make(T, 128, 192, BF)
    full = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    want = torch.autograd.grad(gdn2.gated_feed_forward(*full), full, dy)
    for which in ([0], [1], [2], [3], [1, 2], [0, 3]):
        ins = [t.clone().requires_grad_() if i in which else t for i, t in enumerate((x, wg, wu, wd))]
        got = torch.autograd.grad(gdn2.gated_feed_forward(*ins), [ins[i] for i in which], dy)
        assert all(torch.equal(g, want[i]) for g, i in zip(got, which))
    tied = wg.clone().requires_grad_()                         # one weight in both places: its gradients add up
    g = torch.autograd.grad(gdn2.gated_feed_forward(x, tied, tied, wd), tied, dy)[0]
    o = orc.evaluate(x, wg, wg, wd, "silu", dy)
    both = o["dw_gate"][0] + o["dw_up"][0]
    orc.assert_within(g, both, o["dw_gate"][1] + o["dw_up"][1] + 2**-8 * (o["dw_gate"][0].abs() + o["dw_up"][0].abs()), "dw")


def test_strided_gradient():
    x, wg, wu, wd, _ = make(90, 64, 128, BF)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    grads = torch.autograd.grad(gdn2.gated_feed_forward(*leaves).sum(), leaves)        # an expanded gradient
    want = orc.evaluate(x, wg, wu, wd, "silu", torch.ones(90, 64, device="cuda"))
    for name, g in zip(NAMES, grads):
        orc.assert_within(g, *want[name], name)


def test_gradient_against_differences():
    """Along a direction of w_down, in which y is linear: the difference carries the roundings of the two outputs, half a step each,
    and those of the gradient."""
    x, wg, wu, wd, dy = make(200, 128, 256, F16)
    leaf = wd.clone().requires_grad_()
    g = torch.autograd.grad(gdn2.gated_feed_forward(x, wg, wu, leaf), leaf, dy)[0].double()
    d = torch.randn(wd.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda", dtype=torch.double)
    plus, minus = (wd.double() + 0.25 * d).half(), (wd.double() - 0.25 * d).half()
    yp, ym = (gdn2.gated_feed_forward(x, wg, wu, w).double() for w in (plus, minus))
    diff = ((yp - ym) * dy.double()).sum()
    along = (g * (plus.double() - minus.double())).sum()
    half = 2.0**-11
    tol = half * ((yp.abs() + ym.abs()) * dy.double().abs()).sum() + 3 * half * (g.abs() * (plus.double() - minus.double()).abs()).sum()
    assert abs(float(diff - along)) <= float(tol) and abs(float(along)) > 10 * abs(float(diff - along))


def test_extreme_values():
    """Large pre-activations: the logistic function at its ends, gelu's cube kept finite."""
    for act in ("silu", "gelu_tanh"):
        x = torch.tensor([[3e4], [-3e4], [1e4], [-200.0], [40.0], [-40.0], [0.0]], device="cuda").to(BF).repeat(20, 8)
        wg, wu, wd = torch.eye(8, device="cuda", dtype=BF), torch.eye(8, device="cuda", dtype=BF) * 2**-8, torch.eye(8, device="cuda", dtype=BF)
        check((x, wg, wu, wd, torch.ones(140, 8, device="cuda", dtype=BF)), act)
        x = x[:7]
        y = gdn2.gated_feed_forward(x, wg, wu, wd, act)
        assert torch.isfinite(y).all() and float(y[3].abs().max()) == 0 and float(y[6].abs().max()) == 0


@pytest.mark.parametrize("T", [20, 300])
def test_not_a_number_stays_in_its_row(T):
    x, wg, wu, wd, _ = make(T, 64, 128, BF)
    x[5, 3] = float("nan")
    bad = ~torch.isfinite(gdn2.gated_feed_forward(x, wg, wu, wd))
    assert bad[5].all() and not bad[:5].any() and not bad[6:].any()


@pytest.mark.parametrize("T,hid,inn,out", [(20, 72, 136, 40), (300, 72, 136, 40), (130, 33, 65, 31)])
def test_stays_inside_its_buffers(T, hid, inn, out):
    """Results written between guard rows of a larger allocation."""
    from gdn2_tilelang_b200 import _cabi

    x, wg, wu, wd, dy = make(T, hid, inn, BF, out)
    K = _cabi.kernels()
    ins = K.aligned_rows(x, wg, wu, wd)
    real, made = torch.empty, []

    def guarded(*shape, dtype=None, device=None):
        n = 1
        for s in shape:
            n *= s
        buf = torch.full((n + 512,), 7.0, dtype=dtype, device=device)
        made.append((buf, n))
        return buf[256:256 + n].view(*shape)

    try:
        torch.empty = guarded
        y, kept = K.ffn_forward(*ins, "silu", keep=True)
        grads = K.ffn_backward(*ins, kept, K.aligned_rows(dy)[0], "silu", True, True, True)
    finally:
        torch.empty = real
    torch.cuda.synchronize()
    assert len(made) >= 9
    for buf, n in made:
        assert (buf[:256] == 7).all() and (buf[256 + n:] == 7).all()
    want = orc.evaluate(x, wg, wu, wd, "silu", dy)
    for name, g in zip(NAMES, grads):
        orc.assert_within(g, *want[name], name)
    K.check_device_status()


def test_same_bits_other_stream_and_captured():
    x, wg, wu, wd, dy = make(500, 256, 640, BF)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    y = gdn2.gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2 = gdn2.gated_feed_forward(*leaves)
        grads2 = torch.autograd.grad(y2, leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))
    small = gdn2.gated_feed_forward(x[:3], wg, wu, wd)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inner = [t.detach().requires_grad_() for t in leaves]
        y3 = gdn2.gated_feed_forward(*inner)
        grads3 = torch.autograd.grad(y3, inner, dy)
        with torch.no_grad():
            small3 = gdn2.gated_feed_forward(x[:3], wg, wu, wd)
    for t in (y3.detach(), small3, *grads3):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, y3) and torch.equal(small, small3) and all(torch.equal(a, b) for a, b in zip(grads, grads3))


def test_module_and_a_block_of_both_operators():
    """A gated recurrent residual block as it is trained and decoded: token mixer, channel mixer."""
    torch.manual_seed(0)
    mlp = gdn2.GatedFeedForward(128, 320, "gelu_tanh").cuda().to(BF)
    assert sorted(n for n, _ in mlp.named_parameters()) == ["down_proj.weight", "gate_proj.weight", "up_proj.weight"]
    proj = (torch.randn(3 * 128, 128, device="cuda") * 0.1).to(BF)

    def block(x, mix):
        v, w, g = (x @ proj.t()).split(128, -1)
        x = x + mix(v, -torch.nn.functional.softplus(g.float()), torch.sigmoid(w))
        return x + mlp(x)

    x = torch.randn(2, 75, 128, device="cuda").to(BF).requires_grad_()
    states = []

    def whole(v, g, w):
        o, s = gdn2.gated_recurrence(v, g, w, output_final_state=True)
        states.append(s)
        return o

    y = block(x, whole)
    y.float().square().mean().backward()
    assert x.grad.shape == x.shape and all(torch.isfinite(p.grad).all() and p.grad.any() for p in (x, *mlp.parameters()))
    with torch.no_grad():                                      # the same tokens one by one
        state = torch.zeros(2, 128, device="cuda")
        rows = [block(x[:, t], lambda v, g, w: gdn2.gated_recurrence_step(v, g, w, state)) for t in range(75)]
    # both paths round the same quantities to bf16 at the same places; sums in another order move a rounding by one step, 2^-8 of the
    # value, in x + o (entering the second product, |W| row sums of about 1) and in y: 4 of them
    scale = float(y.detach().abs().max())
    assert float((torch.stack(rows, 1) - y.detach()).abs().max()) <= 4 * 2**-8 * scale
    assert torch.allclose(state, states[0], rtol=0, atol=2**-7 * float(states[0].abs().max()))


@pytest.mark.parametrize("T,hid,inn,out", [(5, 64, 96, 64), (300, 72, 200, 40), (70, 33, 65, 31)])
def test_without_the_host_extension(T, hid, inn, out, monkeypatch):
    from gdn2_tilelang_b200 import _cabi

    ins = make(T, hid, inn, BF, out)
    want = gdn2.gated_feed_forward(*ins[:4])
    monkeypatch.setattr(_cabi.kernels(), "host", None)
    assert torch.equal(gdn2.gated_feed_forward(*ins[:4]), want)
    check(ins, "gelu_tanh")


def test_once_differentiable():
    leaves = [t.requires_grad_() for t in make(9, 8, 16, BF)[:4]]
    grads = torch.autograd.grad(gdn2.gated_feed_forward(*leaves).sum(), leaves[:2], create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        grads[1].sum().backward()


def test_launches_are_counted():
    from gdn2_tilelang_b200 import _cabi

    K = _cabi.kernels()
    x, wg, wu, wd, dy = make(300, 64, 96, BF)
    before = K.launches
    gdn2.gated_feed_forward(x, wg, wu, wd)
    assert K.launches == before + 2
    y = gdn2.gated_feed_forward(x, wg.requires_grad_(), wu, wd)
    y.backward(dy)
    assert K.launches == before + 2 + 2 + 2            # the gated gradient and the pair of weight gradients


def test_offsets_beyond_32_bits():
    """Inner activations of more than 2^31 elements: the last rows against the same tokens alone."""
    T, hid, inn = 400_000, 64, 5632
    x, wg, wu, wd, _ = make(T, hid, inn, BF)
    assert T * inn > 1 << 31
    y = gdn2.gated_feed_forward(x, wg, wu, wd)
    for rows in (slice(0, 300), slice(T - 300, T)):
        orc.assert_within(y[rows], *orc.evaluate(x[rows], wg, wu, wd, "silu")["y"], "y")
    leaf = x.clone().requires_grad_()
    dx = torch.autograd.grad(gdn2.gated_feed_forward(leaf, wg, wu, wd), leaf, torch.ones_like(x))[0]
    for rows in (slice(0, 300), slice(T - 300, T)):
        want = orc.evaluate(x[rows], wg, wu, wd, "silu", torch.ones_like(x[rows]))
        orc.assert_within(dx[rows], *want["dx"], "dx")


@pytest.mark.parametrize("T", [5, 300])
def test_two_streams_at_once(T):
    x, wg, wu, wd, _ = make(T, 512, 1536, BF)
    want = gdn2.gated_feed_forward(x, wg, wu, wd)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(gdn2.gated_feed_forward(x, wg, wu, wd))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in outs)


@pytest.mark.parametrize("T", [40, 127, 300, 1000])
def test_gradients_have_the_same_bits_every_time(T):
    """Nothing is overwritten before it has been read, however the warps' loads and stores queue up."""
    x, wg, wu, wd, dy = make(T, 256, 384, BF)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    first = torch.autograd.grad(gdn2.gated_feed_forward(*leaves), leaves, dy)
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(300):
        for a, b in zip(torch.autograd.grad(gdn2.gated_feed_forward(*leaves), leaves, dy), first):
            differ += (a != b).sum()
    assert int(differ) == 0
