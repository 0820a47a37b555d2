"""``gated_recurrence`` on the GPU against the same recurrence in 64 bits (tolerances: tests/recurrence_oracle.py)."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from tests import recurrence_oracle as orc

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(B, S, D, dtype, gate=True, state=True, seed=0, sequences=None):
    gen = torch.Generator().manual_seed(seed)
    v = torch.randn(B, S, D, generator=gen).to(dtype)
    g = -torch.exp(-6.0 * torch.rand(D, generator=gen)) * torch.rand(B, S, D, generator=gen)
    w = torch.sigmoid(torch.randn(B, S, D, generator=gen)).to(dtype) if gate else None
    s = torch.randn(sequences or B, D, generator=gen) if state else None
    return v, g, w, s


def on_gpu(*ts, grad=False):
    out = [None if t is None else t.cuda() for t in ts]
    if grad:
        for t in out:
            if t is not None:
                t.requires_grad_()
    return out


def check_forward(o, fin, ref):
    ro, rf, eo, ef = ref
    orc.assert_within(o, ro, eo, "o")
    if fin is not None:
        orc.assert_within(fin, rf, ef, "final state")


LENGTHS = [1, 2, 7, 8, 9, 63, 64, 65, 127, 128, 129, 1000, 1025]


@pytest.mark.parametrize("S", LENGTHS)
@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_lengths(S, dtype):
    v, g, w, s = make(2, S, 136, dtype, seed=S)
    o, fin = gdn2.gated_recurrence(*on_gpu(v, g, w, s), output_final_state=True)
    assert o.dtype == dtype and fin.dtype == F32
    check_forward(o, fin, orc.scan(v, g, w, s))


@pytest.mark.parametrize("D", [1, 3, 8, 31, 33, 64, 65, 72, 100, 1001])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("gate", [True, False])
def test_channels(D, dtype, gate):
    v, g, w, s = make(3, 150, D, dtype, gate, state=D % 2 == 0, seed=D)
    o, fin = gdn2.gated_recurrence(*on_gpu(v, g, w, s), output_final_state=True)
    check_forward(o, fin, orc.scan(v, g, w, s))


@pytest.mark.parametrize("B,S,D", [(1, 5000, 64), (1, 3000, 2048), (40, 200, 512), (300, 20, 64)])
def test_clusters_of_every_size(B, S, D):
    v, g, w, s = make(B, S, D, BF, seed=B)
    o, fin = gdn2.gated_recurrence(*on_gpu(v, g, w, s), output_final_state=True)
    check_forward(o, fin, orc.scan(v, g, w, s))
    o2, fin2 = gdn2.gated_recurrence(*on_gpu(v, g, w, s), output_final_state=True)
    assert torch.equal(o, o2) and torch.equal(fin, fin2)          # the same bits on every run
    o3, none = gdn2.gated_recurrence(*on_gpu(v, g, w, s))
    assert none is None and torch.equal(o, o3)


def test_heads_and_trailing_dimensions():
    v, g, w, s = make(2, 70, 96, BF)
    shaped = [t.view(*t.shape[:-1], 4, 24) for t in (v, g, w, s)]
    o, fin = gdn2.gated_recurrence(*on_gpu(*shaped), output_final_state=True)
    assert o.shape == (2, 70, 4, 24) and fin.shape == (2, 4, 24)
    o1, fin1 = gdn2.gated_recurrence(*on_gpu(v, g, w, s), output_final_state=True)
    assert torch.equal(o.flatten(2), o1) and torch.equal(fin.flatten(1), fin1)


@pytest.mark.parametrize("width,first", [(64, 0), (64, 8), (61, 3), (64, 1)])
def test_columns_of_a_projection(width, first):
    """Rows that are columns of a wider tensor, aligned or not, and time-major batches."""
    gen = torch.Generator().manual_seed(4)
    proj = torch.randn(2, 300, 200, generator=gen).to(BF)
    gate = -torch.rand(2, 300, 150, generator=gen)
    cut = lambda p, f: p[..., f:f + width]                          # noqa: E731
    v, w, g = cut(proj, first), cut(proj, first + 100), cut(gate, first)
    pc, gc = proj.cuda(), gate.cuda()
    o, fin = gdn2.gated_recurrence(cut(pc, first), cut(gc, first), cut(pc, first + 100), output_final_state=True)
    check_forward(o, fin, orc.scan(v, g, w, None))
    tm = [t.transpose(0, 1).contiguous().cuda().transpose(0, 1) for t in (v, g, w)]
    o2, fin2 = gdn2.gated_recurrence(*tm, output_final_state=True)
    check_forward(o2, fin2, orc.scan(v, g, w, None))
    sw = [t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in (v, g, w)]     # channels apart: copied
    o3, _ = gdn2.gated_recurrence(*sw)
    check_forward(o3, None, orc.scan(v, g, w, None))
    one = gate[:1, :, first:first + width]                          # one decay for the whole batch, not materialised
    o4, _ = gdn2.gated_recurrence(cut(pc, first), one.cuda().expand(2, -1, -1), cut(pc, first + 100))
    check_forward(o4, None, orc.scan(v, one.expand(2, -1, -1), w, None))


def test_strong_gates():
    """-inf and decays under the smallest normal number forget the state; what follows is exact again."""
    v, g, w, s = make(2, 400, 64, F32)
    g[:, 100], g[0, 101, ::2], g[:, 250], g[1, 399] = float("-inf"), -1e6, -90.0, -103.0
    o, fin = gdn2.gated_recurrence(*on_gpu(v, g, w, s), output_final_state=True)
    check_forward(o, fin, orc.scan(v, g, w, s))
    assert torch.equal(o[:, 100].cpu(), v[:, 100] * w[:, 100])
    zero = torch.zeros_like(g)
    o, _ = gdn2.gated_recurrence(*on_gpu(v, zero, w, s))
    check_forward(o, None, orc.scan(v, zero, w, s))


def test_nan_and_inf_stay_in_their_channel():
    v, g, w, s = make(1, 300, 64, F32)
    v[0, 37, 5], g[0, 50, 9], s[0, 11] = float("nan"), float("nan"), float("inf")
    o, fin = gdn2.gated_recurrence(*on_gpu(v, g, w, s), output_final_state=True)
    bad = ~torch.isfinite(o[0]).cpu()
    assert bad[37:, 5].all() and not bad[:37, 5].any() and bad[50:, 9].all() and not bad[:50, 9].any() and bad[:, 11].all()
    bad[:, [5, 9, 11]] = False
    assert not bad.any()


PACKS = [[0, 5], [0, 0, 1, 1, 3], [0, 64, 128, 193, 500], [0, 0, 700], [0, 300, 300], [0, 1030, 1031, 1100],
         list(range(0, 300))]


@pytest.mark.parametrize("cu", PACKS, ids=lambda c: f"{len(c) - 1}x{c[-1]}")
@pytest.mark.parametrize("D,dtype", [(72, BF), (33, F32)])
def test_packed(cu, D, dtype):
    N = len(cu) - 1
    v, g, w, s = make(1, cu[-1], D, dtype, sequences=N, seed=N)
    vc, gc, wc, sc = on_gpu(v, g, w, s)
    o, fin = gdn2.gated_recurrence(vc, gc, wc, sc, output_final_state=True, cu_seqlens=cu)
    check_forward(o, fin, orc.scan(v, g, w, s, cu))
    o2, fin2 = gdn2.gated_recurrence(vc, gc, wc, sc, output_final_state=True, cu_seqlens=torch.tensor(cu, device="cuda"))
    assert torch.equal(o, o2) and torch.equal(fin, fin2)
    o3, _ = gdn2.gated_recurrence(vc, gc, wc, cu_seqlens=torch.tensor(cu, dtype=torch.int32))
    check_forward(o3, None, orc.scan(v, g, w, None, cu))


def test_no_tokens():
    v, g, w, s = on_gpu(*make(2, 5, 16, BF))
    o, fin = gdn2.gated_recurrence(v[:, :0], g[:, :0], w[:, :0], s, output_final_state=True)
    assert o.shape == (2, 0, 16) and torch.equal(fin, s) and fin.data_ptr() != s.data_ptr()
    assert gdn2.gated_recurrence_decode(v[:, :0], g[:, :0], w[:, :0], s).shape == (2, 0, 16)
    o, fin = gdn2.gated_recurrence(v[:0], g[:0], w[:0], output_final_state=True)
    assert o.shape == (0, 5, 16) and fin.shape == (0, 16)


@pytest.mark.parametrize("n", [1, 2, 5, 8, 9, 200])
@pytest.mark.parametrize("D,dtype", [(128, BF), (33, F16), (33, F32), (36, F32)])
def test_decode(n, D, dtype):
    v, g, w, s = make(5, n, D, dtype, seed=n)
    vc, gc, wc, sc = on_gpu(v, g, w, s)
    where = sc.data_ptr()
    o = gdn2.gated_recurrence_decode(vc, gc, wc, sc)
    ro, rf, eo, ef = orc.scan(v, g, w, s)
    check_forward(o, sc, (ro, rf, eo, ef))
    assert sc.data_ptr() == where
    st = s.cuda()
    rows = [gdn2.gated_recurrence_step(vc[:, t], gc[:, t], wc[:, t], st) for t in range(n)]
    check_forward(torch.stack(rows, 1), st, (ro, rf, eo, ef))


def test_prompt_then_tokens_equal_one_pass():
    v, g, w, s = make(2, 210, 64, BF)
    vc, gc, wc, sc = on_gpu(v, g, w, s)
    o, state = gdn2.gated_recurrence(vc[:, :200], gc[:, :200], wc[:, :200], sc, output_final_state=True)
    outs = [o] + [gdn2.gated_recurrence_decode(vc[:, t:t + 1], gc[:, t:t + 1], wc[:, t:t + 1], state) for t in range(200, 210)]
    check_forward(torch.cat(outs, 1), state, orc.scan(v, g, w, s))


GRADS = [(2, 1, 64, BF), (1, 63, 72, BF), (2, 64, 64, F16), (2, 65, 8, F32), (1, 129, 33, BF), (3, 1001, 101, F32), (1, 1500, 64, BF),
         (24, 130, 512, BF)]


@pytest.mark.parametrize("B,S,D,dtype", GRADS)
@pytest.mark.parametrize("gate", [True, False])
def test_gradients(B, S, D, dtype, gate):
    v, g, w, s = make(B, S, D, dtype, gate, state=S % 2 == 1, seed=S)
    gen = torch.Generator().manual_seed(9)
    do, df = torch.randn(B, S, D, generator=gen).to(dtype), torch.randn(B, D, generator=gen)
    ins = on_gpu(v, g, w, s, grad=True)
    o, fin = gdn2.gated_recurrence(*ins, output_final_state=True)
    check_forward(o, fin, orc.scan(v, g, w, s))
    live = [t for t in ins if t is not None]
    got = dict(zip([n for n, t in zip("vgws", ins) if t is not None], torch.autograd.grad((o, fin), live, (do.cuda(), df.cuda()))))
    want, bound = orc.gradients(v, g, w, s, do, df)
    for name, x, e in zip("vgws", want, bound):
        if name in got:
            orc.assert_within(got[name], x, e, f"d{name}")
    # one gradient only: of the outputs, of the final state
    o, fin = gdn2.gated_recurrence(*ins, output_final_state=True)
    got = torch.autograd.grad(fin, ins[0], df.cuda(), retain_graph=True)[0]
    orc.assert_within(got, *(z[0] for z in orc.gradients(v, g, w, s, None, df)), "dv of the final state")
    got = torch.autograd.grad(o, ins[1], do.cuda())[0]
    orc.assert_within(got, *(z[1] for z in orc.gradients(v, g, w, s, do, None)), "dg of the outputs")


@pytest.mark.parametrize("cu", [[0, 64, 64, 200, 333], [0, 1, 2, 700], list(range(0, 390, 3))], ids=lambda c: f"{len(c) - 1}x{c[-1]}")
def test_packed_gradients(cu):
    N = len(cu) - 1
    v, g, w, s = make(1, cu[-1], 72, BF, sequences=N, seed=N)
    gen = torch.Generator().manual_seed(3)
    do, df = torch.randn(v.shape, generator=gen).to(BF), torch.randn(N, 72, generator=gen)
    ins = on_gpu(v, g, w, s, grad=True)
    o, fin = gdn2.gated_recurrence(*ins, output_final_state=True, cu_seqlens=cu)
    got = torch.autograd.grad((o, fin), ins, (do.cuda(), df.cuda()))
    want, bound = orc.gradients(v, g, w, s, do, df, cu)
    for name, y, x, e in zip("vgws", got, want, bound):
        orc.assert_within(y, x, e, f"d{name}")


def test_gradients_of_shared_and_strided_inputs():
    """One decay for the batch (its gradient is summed by autograd), inputs that are columns of one projection, an expanded
    output gradient."""
    gen = torch.Generator().manual_seed(1)
    proj = torch.randn(2, 100, 128, generator=gen)
    one = -torch.rand(1, 100, 64, generator=gen)
    pc, gc = proj.cuda().requires_grad_(), one.cuda().requires_grad_()
    o, _ = gdn2.gated_recurrence(pc[..., :64], gc.expand(2, -1, -1), pc[..., 64:])
    o.sum().backward()
    v, w, g = proj[..., :64], proj[..., 64:], one.expand(2, -1, -1)
    (dv, dg, dw, _), (ev, eg, ew, _) = orc.gradients(v, g, w, None, torch.ones_like(v), None)
    orc.assert_within(pc.grad, torch.cat([dv, dw], -1), torch.cat([ev, ew], -1), "dproj")
    orc.assert_within(gc.grad, dg.sum(0, keepdim=True), eg.sum(0, keepdim=True) + 2 * orc.U * dg.abs().sum(0, keepdim=True), "dg")


def test_gradients_against_differences():
    """sum(c * o) along a direction. It is linear in v and in w: their differences carry rounding only, 2 * 1e-5 of the terms'
    magnitude over the step; along g the difference formula's own error is h^2 / 6 of the third derivative, bounded by the
    same sum with g's direction to the third power (|d| <= 1: under S^3 of it, so steps are h = 1e-2 / S)."""
    S = 20
    v, g, w, s = (t.cuda() for t in make(1, S, 64, F32))
    gen = torch.Generator().manual_seed(2)
    c = torch.randn(1, S, 64, generator=gen).cuda()
    ins = [t.clone().requires_grad_() for t in (v, g, w, s)]
    o, _ = gdn2.gated_recurrence(*ins)
    grads = torch.autograd.grad(o, ins, c)

    def f(vals):
        return (gdn2.gated_recurrence(*vals)[0].double() * c.double()).sum()

    magnitude = orc.scan(v.abs().cpu(), g.cpu(), w.cpu(), s.abs().cpu())[0].sum() * float(c.abs().max())
    for i, step in enumerate((1.0, 1e-2 / S, 1.0, 1.0)):
        d = torch.rand(ins[i].shape, generator=gen).cuda() * 2 - 1
        plus, minus = ([t.clone() for t in (v, g, w, s)] for _ in range(2))
        plus[i] += step * d
        minus[i] -= step * d
        diff = (f(plus) - f(minus)) / (2 * step)
        along = (grads[i].double() * d.double()).sum()
        tol = 20 * orc.STEP * float(magnitude) * 4 / step + (step**2 * S**3 * float(magnitude) if i == 1 else 0)
        assert abs(float(diff - along)) <= tol, (i, float(diff), float(along), tol)


def test_stays_inside_its_buffers():
    """Rows before and behind the inputs, and what the allocator put around outputs, are left alone: a slice of a longer batch
    gives the bits of the slice alone, whatever stands around it."""
    v, g, w, s = on_gpu(*make(2, 300, 72, BF))
    o, fin = gdn2.gated_recurrence(v[:, 50:171].contiguous(), g[:, 50:171].contiguous(), w[:, 50:171].contiguous(), s, True)
    v2, g2, w2 = v.clone(), g.clone(), w.clone()
    for t in (v2, g2, w2):
        t[:, :50], t[:, 171:] = float("nan"), float("nan")
    o2, fin2 = gdn2.gated_recurrence(v2[:, 50:171], g2[:, 50:171], w2[:, 50:171], s, True)
    assert torch.equal(o, o2) and torch.equal(fin, fin2)


def test_another_stream_and_a_captured_call():
    v, g, w, s = on_gpu(*make(2, 500, 128, BF))
    want, wfin = gdn2.gated_recurrence(v, g, w, s, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o, fin = gdn2.gated_recurrence(v, g, w, s, True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, want) and torch.equal(fin, wfin)
    graph = torch.cuda.CUDAGraph()
    do = torch.randn_like(v)
    leaves = [t.clone().requires_grad_() for t in (v, g, w, s)]
    ref = torch.autograd.grad(gdn2.gated_recurrence(*leaves)[0], leaves, do)
    with torch.cuda.graph(graph):
        o, fin = gdn2.gated_recurrence(v, g, w, s, True)
        inner = [t.detach().requires_grad_() for t in leaves]
        grads = torch.autograd.grad(gdn2.gated_recurrence(*inner)[0], inner, do)
    for t in (o, fin, *grads):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, want) and torch.equal(fin, wfin)
    assert all(torch.equal(a, b) for a, b in zip(grads, ref))


def test_a_long_sequence():
    """2^17 tokens: products of decays over the whole of it, two channel groups, the state at the end."""
    S, D = 1 << 17, 72
    gen = torch.Generator(device="cuda").manual_seed(0)
    v = torch.randn(1, S, D, generator=gen, device="cuda")
    g = -1e-3 * torch.rand(1, S, D, generator=gen, device="cuda")
    o, fin = gdn2.gated_recurrence(v, g, output_final_state=True)
    # the last 40000 tokens in 64 bits from the kernel's own state before them: what came before has decayed by e^-20
    lo = S - 40000
    h = o[0, lo - 1].double()
    G = g[0, lo:].double().cumsum(0)
    want = ((G[-1] - G).exp() * v[0, lo:].double()).sum(0) + G[-1].exp() * h
    # memory of 2000 tokens, 8 u a step of a magnitude of 2000 * 0.8: STEP * 2000 * 1600
    for got in (fin[0], o[0, -1]):
        assert float((got.double() - want).abs().max()) <= orc.STEP * 2000 * 1600


@pytest.fixture
def through_python(monkeypatch):
    """Without the host extension every call goes through Python."""
    from gdn2_tilelang_b200 import _cabi

    monkeypatch.setattr(_cabi.kernels(), "host", None)


@pytest.mark.parametrize("B,S,D,dtype", GRADS[:3] + GRADS[4:5])
def test_without_the_host_extension(B, S, D, dtype, through_python):
    test_gradients(B, S, D, dtype, True)
    test_decode(3, D, dtype)
    test_packed([0, 5, 5, 70], D, dtype)


def test_once_differentiable():
    v, g, w, s = on_gpu(*make(1, 9, 8, F32), grad=True)
    grads = torch.autograd.grad(gdn2.gated_recurrence(v, g, w, s)[0].sum(), (v, g), create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        grads[1].sum().backward()


def test_launches_are_counted():
    from gdn2_tilelang_b200 import _cabi

    K = _cabi.kernels()
    v, g, w, s = on_gpu(*make(1, 9, 8, F32), grad=True)
    before = K.launches
    o, _ = gdn2.gated_recurrence(v, g, w, s)
    assert K.launches == before + 1
    o.sum().backward()
    assert K.launches == before + 2


def test_offsets_beyond_32_bits():
    """More than 2^31 elements an input. Memory is 20 tokens here: the last rows from zero, 3000 tokens before them, to 32 bits."""
    S, D = (1 << 21) + 77, 1032
    gen = torch.Generator(device="cuda").manual_seed(0)
    v = torch.empty(1, S, D, dtype=BF, device="cuda").normal_(generator=gen)
    g = torch.full((1, S, D), -0.05, device="cuda")
    assert v.numel() > 1 << 31
    o, fin = gdn2.gated_recurrence(v, g, output_final_state=True)
    lo = S - 4000
    tail, tfin = gdn2.gated_recurrence(v[:, lo:], g[:, lo:], output_final_state=True)
    # 3000 tokens of exp(-0.05) leave e^-150 of what came before: the same sums but for the order they are composed in
    mag = orc.STEP * 20 * 20 * 5                                   # 8 u a step, a memory and a magnitude of 20 and |v| < 5
    assert float((fin - tfin).abs().max()) <= 2 * mag
    assert float((o[:, lo + 3000:].float() - tail[:, 3000:].float()).abs().max()) <= 2 * mag + 2**-8 * 20
    del o, tail
    do = torch.ones(1, 1, 1, dtype=BF, device="cuda").expand(1, S, D)
    leaf = v.requires_grad_()
    out, _ = gdn2.gated_recurrence(leaf, g)
    dv = torch.autograd.grad(out, leaf, do)[0]
    a = float(torch.tensor(-0.05, dtype=torch.float64).exp())
    assert torch.all(dv[0, -1] == 1) and torch.all(dv[0, 0] == dv[0, 5000]) and abs(float(dv[0, 0, 0]) - 1 / (1 - a)) <= 2**-8 / (1 - a)


def test_two_streams_at_once():
    v, g, w, s = on_gpu(*make(2, 3000, 512, BF))
    want = gdn2.gated_recurrence(v, g, w, s, True)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(gdn2.gated_recurrence(v, g, w, s, True))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[0]) and torch.equal(f, want[1]) for o, f in outs)


def test_other_types_of_decay_and_state():
    v, g, w, s = make(2, 40, 64, BF)
    g, s = g.to(BF), s.to(F16)
    vc, gc, wc, sc = on_gpu(v, g, w, s, grad=True)
    o, fin = gdn2.gated_recurrence(vc, gc, wc, sc, output_final_state=True)
    check_forward(o, fin, orc.scan(v, g, w, s))
    dg, ds = torch.autograd.grad(o.float().sum(), (gc, sc))
    assert dg.dtype == BF and ds.dtype == F16
    (_, want, _, wantds), (_, eg, _, es) = orc.gradients(v, g, w, s, torch.ones_like(v), None)
    orc.assert_within(dg, want, eg, "dg")
    orc.assert_within(ds, wantds, es, "dstate")


@pytest.mark.parametrize("B,S,D", [(2, 700, 512), (1, 5000, 64), (3, 333, 2048), (1, 4097, 33)])
def test_gradients_have_the_same_bits_every_time(B, S, D):
    ins = on_gpu(*make(B, S, D, BF), grad=True)
    do = torch.randn(B, S, D, device="cuda").to(BF)
    first = torch.autograd.grad(gdn2.gated_recurrence(*ins)[0], ins, do)
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(200):
        for a, b in zip(torch.autograd.grad(gdn2.gated_recurrence(*ins)[0], ins, do), first):
            differ += (a != b).sum()
    assert int(differ) == 0
