"""``gated_recurrence``'s refusals and the C entry points' checks (no GPU), and the oracle against differences."""

from __future__ import annotations

import ctypes

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from gdn2_tilelang_b200 import _cabi
from tests import recurrence_oracle as orc


@pytest.fixture
def any_device(monkeypatch):
    """Host tensors pass the device check, so that the checks behind it are reached; no kernel may be."""
    monkeypatch.setattr(_cabi, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(_cabi, "kernels", lambda: pytest.fail("a refused call reached the kernels"))


def rows(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA devices only"):
        gdn2.gated_recurrence(rows(1, 4, 8), rows(1, 4, 8))
    with pytest.raises(ValueError, match="CUDA devices only"):
        gdn2.gated_recurrence_decode(rows(1, 4, 8), rows(1, 4, 8), None, rows(1, 8))


def test_refusals(any_device):
    v, g = rows(2, 4, 8), rows(2, 4, 8)
    for bad in (dict(v=rows(4, 8)), dict(g=rows(2, 4, 9)), dict(w=rows(2, 5, 8)), dict(initial_state=rows(2, 9)),
                dict(initial_state=rows(1, 8)), dict(cu_seqlens=[0, 4])):
        with pytest.raises(ValueError):
            gdn2.gated_recurrence(**{"v": v, "g": g, **bad})
    for bad in (dict(v=rows(2, 4, 8, dtype=torch.float64)), dict(w=rows(2, 4, 8, dtype=torch.bfloat16)),
                dict(g=rows(2, 4, 8, dtype=torch.int32)), dict(initial_state=rows(2, 8, dtype=torch.int64))):
        with pytest.raises(TypeError):
            gdn2.gated_recurrence(**{"v": v, "g": g, **bad})
    one = rows(1, 4, 8)
    for cu in ([0], [0, 3], [1, 4], [0, 3, 2, 4], [0, 5], []):
        with pytest.raises(ValueError, match="cu_seqlens"):
            gdn2.gated_recurrence(one, one, cu_seqlens=cu)
    with pytest.raises(ValueError, match="shape"):
        gdn2.gated_recurrence(one, one, initial_state=rows(1, 8), cu_seqlens=torch.tensor([0, 2, 4]))


def test_decode_refusals(any_device):
    v = rows(2, 1, 8)
    with pytest.raises(ValueError, match="shape"):
        gdn2.gated_recurrence_decode(v, v, v, rows(2, 9))
    with pytest.raises(ValueError, match="float32"):
        gdn2.gated_recurrence_decode(v, v, v, rows(2, 8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="contiguous"):
        gdn2.gated_recurrence_decode(v, v, v, rows(8, 2).t())
    with pytest.raises(ValueError, match="no gradient"):
        gdn2.gated_recurrence_decode(v, v, v, rows(2, 8).requires_grad_())
    with pytest.raises(ValueError):
        gdn2.gated_recurrence_step(rows(8), rows(8), None, rows(8))


def args(**kw):
    a = _cabi.RecurrenceArgs(v=16, g=16, o=16, sequences=1, B=1, S=4, D=8)
    for k, x in kw.items():
        setattr(a, k, x)
    return ctypes.byref(a)


def test_c_entry_checks():
    lib = _cabi.load_library()
    f, b = lib.gdn2_recurrence_forward, lib.gdn2_recurrence_backward
    assert f(None, 0, None) == -1 and b(None, 0, None) == -1
    assert f(args(), 9, None) == -3
    assert f(args(v=None), 0, None) == -1 and f(args(g=None), 0, None) == -1 and f(args(o=None), 0, None) == -1
    assert b(args(), 0, None) == -1
    grads = dict(dout=16, dv=16, dg=16, marks=16)
    assert b(args(w=16, **grads), 0, None) == -1                   # a gate without room for its gradient
    for kw in (dict(B=0), dict(S=0), dict(D=0), dict(S=1 << 31), dict(v_token_stride=-1), dict(g_batch_stride=-8)):
        assert f(args(**kw), 0, None) == -2
        assert b(args(**kw, **grads), 0, None) == -2
    cu = lambda *x: (ctypes.c_int64 * len(x))(*x)                  # noqa: E731
    for c, n, B in ((cu(0, 3), 1, 1), (cu(1, 4), 1, 1), (cu(0, 3, 2, 4), 3, 1), (cu(0, 4), 1, 2), (cu(0, 4), 0, 1)):
        assert f(args(cu_seqlens=c, sequences=n, B=B), 0, None) == -2


def test_marks():
    lib = _cabi.load_library()
    n = lib.gdn2_recurrence_marks
    assert n(3, 64, None, 3) == 3 and n(3, 65, None, 3) == 6 and n(1, 1, None, 1) == 1
    cu = (ctypes.c_int64 * 5)(0, 0, 1, 65, 130)
    assert n(1, 130, cu, 4) == 0 + 1 + 1 + 2


def test_oracle_gradient_against_autograd():
    gen = torch.Generator().manual_seed(0)
    v, w, do = (torch.randn(2, 9, 5, generator=gen, dtype=torch.float64) for _ in range(3))
    g = -torch.rand(2, 9, 5, generator=gen, dtype=torch.float64)
    s, df = torch.randn(2, 5, generator=gen, dtype=torch.float64), torch.randn(2, 5, generator=gen, dtype=torch.float64)
    ins = [t.requires_grad_() for t in (v, g, w, s)]
    h, outs = s, []
    for t in range(9):
        h = torch.exp(g[:, t]) * h + w[:, t] * v[:, t]
        outs.append(h)
    o = torch.stack(outs, 1)
    want = torch.autograd.grad((o, h), ins, (do, df))
    got, _ = orc.gradients(v, g, w, s, do, df)
    assert torch.allclose(orc.scan(v, g, w, s)[0], o.detach())
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)
