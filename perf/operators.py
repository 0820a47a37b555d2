"""The operators of a gated recurrent block this package is timed on, and their plain forms.

Two operators, each with the gradient a training step needs and the form a token-by-token server needs:

    gated_recurrence    h_t = exp(g_t) * h_{t-1} + w_t * v_t per channel, o_t = h_t: the diagonal recurrence that stacks of
                        recurrent layers put beside gated delta layers. g is the float32 natural-log decay (<= 0), w an
                        optional write gate, the state float32. Whole sequences, packed sequences, single tokens in place.
    gated_feed_forward  y = (act(x Wg^T) * (x Wu^T)) Wd^T: the channel mixer after every token mixer.

A case is a dict of plain values. ``kind`` is the call it makes:

    scan        ``gated_recurrence`` over a batch, optionally continuing from a state
    scan_packed the same with ``cu_seqlens``: sequences of unequal lengths in one row
    scan_train  the same with gradients of every input for given gradients of o and of the final state
    decode      ``gated_recurrence_decode``: n tokens, the state updated in place
    ffn         ``gated_feed_forward`` of ``tokens`` tokens
    ffn_train   the same with gradients of x and of the three weights
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one token of one conversation: the latency of the call itself
        _scan("scan_step_b1", "decode", B=1, S=1),
        # one token for each of 256 conversations, the decode batch of the benchmark
        _scan("scan_step_b256", "decode", B=256, S=1),
        # two prompts of the layer benchmark's length, continuing from a state
        _scan("scan_prompts", "scan", B=2, S=4096, state=True),
        # one long document, fewer channels, half precision, a length that no tile divides
        _scan("scan_document_f16", "scan", B=1, S=65573, D=1024, dtype="f16"),
        # ten prompts of unequal lengths packed into one row
        _scan("scan_packed", "scan_packed", B=1, S=16037, seqs=10, lengths=1),
        # a training step's forward and backward
        _scan("scan_train", "scan_train", B=4, S=4096, state=True),
        # full precision, odd sizes, no write gate
        _scan("scan_train_f32_odd", "scan_train", B=3, S=1001, D=1001, dtype="f32", write_gate=False),
        # one token of one conversation through the feed-forward: the weights are read once
        _ffn("ffn_step_b1", "ffn", tokens=1),
        # one token for each of 24 conversations, half precision
        _ffn("ffn_step_b24_f16", "ffn", tokens=24, dtype="f16"),
        # the layer benchmark's two prompts of 4096 tokens
        _ffn("ffn_prompts", "ffn", tokens=8192),
        # odd sizes throughout, the other activation
        _ffn("ffn_odd_gelu", "ffn", tokens=1003, hidden=1001, inner=2731, activation="gelu_tanh"),
        # a training step's forward and backward
        _ffn("ffn_train", "ffn_train", tokens=8192),
    ]


def _scan(name, kind, B, S, D=2048, dtype="bf16", write_gate=True, state=False, seqs=1, lengths=0):
    return dict(name=name, kind=kind, B=B, S=S, D=D, dtype=dtype, write_gate=write_gate, state=state, seqs=seqs,
                lengths=lengths)


def _ffn(name, kind, tokens, hidden=2048, inner=5632, activation="silu", dtype="bf16"):
    return dict(name=name, kind=kind, tokens=tokens, hidden=hidden, inner=inner, activation=activation, dtype=dtype)


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["scan", "scan", "scan_packed", "scan_train", "scan_train", "decode", "ffn", "ffn", "ffn_train",
                       "ffn_train"])
    dtype = rng.choice(["bf16", "bf16", "f16"] if kind.startswith("ffn") else ["bf16", "bf16", "f16", "f32"])
    if kind.startswith("ffn"):
        hidden, inner = _log_uniform(rng, 200, 2048), _log_uniform(rng, 300, 5632)
        if rng.random() < 0.7:                                                       # most models have even-handed sizes
            hidden, inner = -(-hidden // 64) * 64, -(-inner // 64) * 64
        tokens = _log_uniform(rng, 1 if kind == "ffn" else 16, 8192)
        case = _ffn("", kind, tokens, hidden, inner, rng.choice(["silu", "silu", "gelu_tanh"]), dtype)
    else:
        D = _log_uniform(rng, 64, 4096)
        if rng.random() < 0.7:
            D = -(-D // 32) * 32
        gate, state = rng.random() < 0.7, rng.random() < 0.5
        if kind == "decode":
            case = _scan("", kind, _log_uniform(rng, 1, 256), rng.choice([1, 1, 1, 2, 3, 5, 8]), D, dtype, gate, True)
        elif kind == "scan_packed":
            seqs = rng.randint(2, 40)
            case = _scan("", kind, 1, _log_uniform(rng, 2 * seqs, 32000000 // max(D, 1000)), D, dtype, gate, state, seqs,
                         rng.randint(1, 10**6))
        else:
            B = rng.choice([1, 1, 2, 3, 4, 8])
            most = 32000000 // (B * max(D, 500))
            case = _scan("", kind, B, _log_uniform(rng, 1, most), D, dtype, gate, state)
    del case["name"]
    return case


def _sequence_offsets(case):
    """``cu_seqlens`` of a packed case: the token axis cut at random places; two cuts may fall together."""
    rng = random.Random(case["lengths"])
    return [0] + sorted(rng.randint(0, case["S"]) for _ in range(case["seqs"] - 1)) + [case["S"]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    st = {"case": case}
    train = case["kind"].endswith("_train")
    if case["kind"].startswith("ffn"):
        T, hid, inn = case["tokens"], case["hidden"], case["inner"]
        st["x"] = normal(T, hid).to(dt)
        for name, rows, cols in (("w_gate", inn, hid), ("w_up", inn, hid), ("w_down", hid, inn)):
            st[name] = (normal(rows, cols) * cols**-0.5).to(dt)
        if train:
            st["dy"] = normal(T, hid).to(dt)
            for name in ("x", "w_gate", "w_up", "w_down"):
                st[name].requires_grad_()
        return st
    B, S, D = case["B"], case["S"], case["D"]
    seqs = case["seqs"] if case["kind"] == "scan_packed" else B
    st["v"] = normal(B, S, D).to(dt)
    # decays from a few tokens to thousands of them, a scale per channel
    st["g"] = -torch.exp(-7.0 * torch.rand(D, generator=gen, device="cuda")) * torch.sigmoid(normal(B, S, D))
    st["w"] = torch.sigmoid(normal(B, S, D)).to(dt) if case["write_gate"] else None
    st["state"] = normal(seqs, D) if case["state"] or case["kind"] == "decode" else None
    if case["kind"] == "scan_packed":
        st["cu_seqlens"] = torch.tensor(_sequence_offsets(case), dtype=torch.int32)      # a scheduler has the lengths on the host
    if train:
        st["do"], st["dfinal"] = normal(B, S, D).to(dt), normal(seqs, D)
        for name in ("v", "g", "w", "state"):
            if st[name] is not None:
                st[name].requires_grad_()
    return st


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        import gdn2_tilelang_b200 as gdn2

        if kind == "decode":
            return gdn2.gated_recurrence_decode(state["v"], state["g"], state["w"], state["state"]), state["state"]
        if kind == "scan":
            return gdn2.gated_recurrence(state["v"], state["g"], state["w"], state["state"], output_final_state=True)
        if kind == "scan_packed":
            return gdn2.gated_recurrence(state["v"], state["g"], state["w"], state["state"], output_final_state=True,
                                         cu_seqlens=state["cu_seqlens"])
        if kind == "scan_train":
            ins = [state[n] for n in ("v", "g", "w", "state")]
            o, final = gdn2.gated_recurrence(*ins, output_final_state=True)
            grads = torch.autograd.grad((o, final), [t for t in ins if t is not None], (state["do"], state["dfinal"]))
            return o.detach(), final.detach(), list(grads)
        ins = [state[n] for n in ("x", "w_gate", "w_up", "w_down")]
        y = gdn2.gated_feed_forward(*ins, activation=case["activation"])
        if kind == "ffn":
            return y
        return y.detach(), list(torch.autograd.grad(y, ins, state["dy"]))
    with torch.no_grad():
        return (_plain_ffn if kind.startswith("ffn") else _plain_scan)(state)


def _rows_from(a, x):
    """All h_t = a_t * h_{t-1} + x_t (h before the first row is zero) along dimension 1, by doubling."""
    a, x, d, S = a.clone(), x.clone(), 1, x.shape[1]
    while d < S:
        x[:, d:] = x[:, d:] + a[:, d:] * x[:, :-d]
        a[:, d:] = a[:, d:] * a[:, :-d]
        d *= 2
    return x


def _plain_scan(state):
    # in 64 bits: a decay near 1 that is off by a hundredth of a 32-bit step tells after thousands of tokens
    case, dt = state["case"], DTYPES[state["case"]["dtype"]]
    v, g = state["v"].double(), state["g"].double()
    w = state["w"].double() if state["w"] is not None else None
    decay, h0 = torch.exp(g), state["state"]
    x = v if w is None else w * v
    if case["kind"] == "scan_packed":
        cu = state["cu_seqlens"].to(v.device, torch.int64)
        lo, some = cu[:-1], cu[1:] > cu[:-1]
        x, first = x.clone(), lo[some]
        if h0 is not None:
            x[0, first] = x[0, first] + decay[0, first] * h0[some]
        decay = decay.clone()
        decay[0, first] = 0.0
        h = _rows_from(decay, x)
        last = (cu[1:] - 1).clamp(min=0)
        before = torch.zeros_like(h[0, last]) if h0 is None else h0
        return h.to(dt), torch.where(some[:, None], h[0, last], before).float()
    if h0 is not None:
        x = torch.cat([x[:, :1] + decay[:, :1] * h0[:, None], x[:, 1:]], 1)
    h = _rows_from(decay, x)
    if case["kind"] == "decode":
        h0.copy_(h[:, -1])
        return h.to(dt), h0
    final = h[:, -1].float()
    if case["kind"] == "scan":
        return h.to(dt), final
    do = state["do"].double()
    do = torch.cat([do[:, :-1], do[:, -1:] + state["dfinal"][:, None]], 1)
    # dh_t = do_t + exp(g_{t+1}) * dh_{t+1}: the same rows from the other end
    later = torch.cat([decay[:, 1:], torch.zeros_like(decay[:, :1])], 1)
    dh = _rows_from(later.flip(1), do.flip(1)).flip(1)
    start = torch.zeros_like(h[:, 0]) if h0 is None else h0.double()
    before = torch.cat([start[:, None], h[:, :-1]], 1)
    grads = [dh.to(dt) if w is None else (dh * w).to(dt), (dh * decay * before).float()]
    if w is not None:
        grads.append((dh * v).to(dt))
    if h0 is not None:
        grads.append((decay[:, 0] * dh[:, 0]).float())
    return h.to(dt), final, grads


def _plain_ffn(state):
    case, dt = state["case"], DTYPES[state["case"]["dtype"]]
    x, wg, wu, wd = (state[n].float() for n in ("x", "w_gate", "w_up", "w_down"))
    a, u = x @ wg.T, x @ wu.T
    if case["activation"] == "silu":
        s = 1.0 / (1.0 + torch.exp(-a))
        act, slope = a * s, s * (1.0 + a * (1.0 - s))
    else:
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (a + 0.044715 * a * a * a))
        act = 0.5 * a * (1.0 + t)
        slope = 0.5 * (1.0 + t) + 0.5 * a * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * a * a)
    h = act * u
    y = (h @ wd.T).to(dt)
    if case["kind"] == "ffn":
        return y
    dy = state["dy"].float()
    dh = dy @ wd
    da, du = dh * u * slope, dh * act
    return y, [(da @ wg + du @ wu).to(dt), (da.T @ x).to(dt), (du.T @ x).to(dt), (dy.T @ h).to(dt)]


def exact(case, seed):
    """The definitions token by token and product by product in 64 bits."""
    st = {k: v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in prepare(case, seed).items()}
    if case["kind"].startswith("ffn"):
        x, wg, wu, wd = (st[n] for n in ("x", "w_gate", "w_up", "w_down"))
        a, u = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
        if case["activation"] == "silu":
            act, slope = a * torch.sigmoid(a), torch.sigmoid(a) + a * torch.sigmoid(a) * torch.sigmoid(-a)
        else:
            k = (2.0 / math.pi) ** 0.5
            inner, dinner = k * a * (1.0 + 0.044715 * a.square()), k * (1.0 + 0.134145 * a.square())
            act = a * (1.0 + torch.tanh(inner)) / 2.0
            slope = (1.0 + torch.tanh(inner)) / 2.0 + a / 2.0 * dinner / torch.cosh(inner).square()
        y = torch.matmul(act * u, wd.t())
        if case["kind"] == "ffn":
            return y
        dh = torch.matmul(st["dy"], wd)
        dgate, dup = dh * u * slope, dh * act
        return y, [torch.matmul(dgate, wg) + torch.matmul(dup, wu), torch.matmul(dgate.t(), x), torch.matmul(dup.t(), x),
                   torch.matmul(st["dy"].t(), act * u)]
    B, S, D = case["B"], case["S"], case["D"]
    v, g, w = st["v"], st["g"], st["w"]
    bounds = _sequence_offsets(case) if case["kind"] == "scan_packed" else [0, S]
    seqs = len(bounds) - 1
    o = torch.empty(B, S, D, dtype=torch.float64, device=v.device)
    final = torch.empty(seqs if seqs > 1 else B, D, dtype=torch.float64, device=v.device)
    for i, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        rows = slice(i, i + 1) if seqs > 1 else slice(None)
        h = torch.zeros_like(final[rows]) if st["state"] is None else st["state"][rows]
        for t in range(lo, hi):
            h = torch.exp(g[:, t]) * h + (v[:, t] if w is None else w[:, t] * v[:, t])
            o[:, t] = h
        final[rows] = h
    if case["kind"] != "scan_train":
        return o, final
    dv, dg, dw = torch.empty_like(o), torch.empty_like(o), torch.empty_like(o)
    start = torch.zeros_like(final) if st["state"] is None else st["state"]
    dh = st["dfinal"]
    for t in range(S - 1, -1, -1):
        dh = dh + st["do"][:, t]
        dv[:, t] = dh if w is None else dh * w[:, t]
        dw[:, t] = dh * v[:, t]
        into = torch.exp(g[:, t]) * dh
        dg[:, t] = into * (o[:, t - 1] if t else start)
        dh = into
    return o, final, [dv, dg] + ([] if w is None else [dw]) + ([] if st["state"] is None else [dh])


def work(case):
    """Each input once and each output once; two operations per multiply-add of the projections, and of the recurrence the
    decay's exponential as one operation, the write gate's product and the update."""
    e = BYTES[case["dtype"]]
    if case["kind"].startswith("ffn"):
        T, hid, inn = case["tokens"], case["hidden"], case["inner"]
        weights, rows = 3 * hid * inn * e, T * hid * e
        if case["kind"] == "ffn":
            return {"bytes": weights + 2 * rows, "flops": 6.0 * T * hid * inn}
        return {"bytes": 2 * weights + 4 * rows, "flops": 18.0 * T * hid * inn}
    B, S, D = case["B"], case["S"], case["D"]
    gates = 1 if case["write_gate"] else 0
    states = 4 * D * (case["seqs"] if case["kind"] == "scan_packed" else B)
    n = B * S * D
    bytes_ = n * (e * (2 + gates) + 4) + states * (2 if case["state"] or case["kind"] == "decode" else 1)
    flops = n * (3.0 + gates)
    if case["kind"] == "scan_train":                  # the backward pass reads do beside the inputs and writes their gradients
        bytes_ += n * (e * (2 + gates) + 4) + states * (2 if case["state"] else 1)
        flops += n * (5.0 + 2 * gates)
    return {"bytes": float(bytes_), "flops": flops}
