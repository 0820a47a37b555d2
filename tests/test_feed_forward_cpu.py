"""``gated_feed_forward``'s refusals, the C entry points' checks and the oracle against autograd (no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from gdn2_tilelang_b200 import _cabi
from tests import ffn_oracle as orc

BF = torch.bfloat16


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA devices only"):
        gdn2.gated_feed_forward(z(3, 8), z(16, 8), z(16, 8), z(8, 16))


def test_refusals(monkeypatch):
    monkeypatch.setattr(_cabi, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(_cabi, "kernels", lambda: pytest.fail("a refused call reached the kernels"))
    ok = dict(x=z(3, 8), w_gate=z(16, 8), w_up=z(16, 8), w_down=z(8, 16))
    for bad in (dict(x=z(3, 9)), dict(w_up=z(17, 8)), dict(w_gate=z(17, 8)), dict(w_down=z(8, 17)), dict(w_down=z(8)),
                dict(x=z(())), dict(activation="relu"), dict(w_down=z(0, 16)),
                dict(w_gate=z(0, 8), w_up=z(0, 8), w_down=z(8, 0)), dict(x=z(3, 0), w_gate=z(16, 0), w_up=z(16, 0))):
        with pytest.raises(ValueError):
            gdn2.gated_feed_forward(**{**ok, **bad})
    for bad in (dict(x=z(3, 8, dtype=torch.float16)), {k: t.float() for k, t in ok.items()}, dict(w_down=z(8, 16, dtype=torch.float32))):
        with pytest.raises(TypeError):
            gdn2.gated_feed_forward(**{**ok, **bad})
    with pytest.raises(ValueError, match="activation"):
        gdn2.GatedFeedForward(8, 16, "tanh")


def args(**kw):
    a = _cabi.FfnArgs(x=16, w_gate=16, w_up=16, w_down=16, h=16, y=16, tokens=4, hidden=8, inner=16, out=8, x_stride=8, w_gate_stride=8,
                      w_up_stride=8, w_down_stride=16, inner_stride=16, y_stride=8, dy_stride=8, dx_stride=8)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_c_entry_checks():
    lib = _cabi.load_library()
    f, b = lib.gdn2_ffn_forward, lib.gdn2_ffn_backward
    kept = dict(kept=16, dy=16, da=16, du=16, dx=16)
    assert f(None, 1, None) == -1 and b(None, 1, None) == -1
    assert f(args(), 0, None) == -3 and b(args(**kept), 0, None) == -3 and f(args(), 7, None) == -3
    assert f(args(activation=2), 1, None) == -8
    for name in ("x", "w_gate", "w_up", "w_down", "h", "y"):
        assert f(args(**{name: None}), 1, None) == -1
    for name in ("dy", "kept", "da", "du"):
        assert b(args(**{**kept, name: None}), 1, None) == -1
    assert b(args(**kept, dw_gate=16), 1, None) == -1                      # dw_gate without dw_up
    for bad in (dict(tokens=0), dict(hidden=0), dict(inner=-1), dict(out=0), dict(tokens=1 << 31), dict(x_stride=0), dict(w_down_stride=8),
                dict(inner_stride=8), dict(tokens=1 << 29, inner=1 << 20, inner_stride=1 << 20, w_down_stride=1 << 20)):
        assert f(args(**bad), 1, None) == -2
        assert b(args(**kept, **bad), 1, None) == -2
    assert f(args(y_stride=7), 1, None) == -2 and b(args(**kept, dy_stride=7), 1, None) == -2 and b(args(**{**kept}, dx_stride=7), 1, None) == -2
    for bad in (dict(x=24), dict(w_up=8), dict(x_stride=12), dict(w_down_stride=17), dict(inner_stride=17), dict(inner_stride=24)):
        assert f(args(**bad), 1, None) == -4
        assert b(args(**kept, **bad), 1, None) == -4
    assert b(args(**{**kept, "dy": 24}), 1, None) == -4


def test_row_copy_checks():
    lib = _cabi.load_library()
    g = lib.gdn2_align_rows
    copy = lambda *a: ctypes.byref(_cabi.RowCopy(*a))                      # noqa: E731
    assert g(None, 1, None) == -1
    assert g(copy(2, 16, 1, 1, 0, 8), 0, None) == -2 and g(copy(2, 16, 1, 1, 0, 8), 7, None) == -2
    assert g(copy(None, 16, 1, 1, 0, 8), 1, None) == -1 and g(copy(2, None, 1, 1, 0, 8), 1, None) == -1
    assert g(copy(2, 16, 0, 1, 0, 8), 1, None) == -2 and g(copy(2, 16, 1, 9, 0, 8), 1, None) == -2
    assert g(copy(2, 24, 1, 1, 0, 8), 1, None) == -4 and g(copy(2, 16, 1, 1, 0, 9), 1, None) == -4


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_oracle_against_autograd(act):
    gen = torch.Generator().manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=gen).to(BF)                   # noqa: E731
    x, wg, wu, wd, dy = n(5, 7), n(11, 7), n(11, 7), n(6, 11), n(5, 6)
    leaves = [t.double().requires_grad_() for t in (x, wg, wu, wd)]
    a, u = leaves[0] @ leaves[1].T, leaves[0] @ leaves[2].T
    f = torch.nn.functional.silu(a) if act == "silu" else torch.nn.functional.gelu(a, approximate="tanh")
    y = (f * u) @ leaves[3].T
    grads = torch.autograd.grad(y, leaves, dy.double())
    got = orc.evaluate(x, wg, wu, wd, act, dy)
    for name, want in zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), (y.detach(), *grads)):
        assert torch.allclose(got[name][0], want, rtol=1e-12, atol=1e-12), name


def test_rows_that_need_no_copy(monkeypatch):
    """What is aligned goes as it is; the rest is copied in one launch, to a pitch of 16 bytes."""
    calls = []

    class Lib:
        def gdn2_align_rows(self, copies, n, stream):
            calls.append([(c.rows, c.cols, c.src_stride, c.dst_stride) for c in copies])
            return 0

    K = _cabi.NativeKernels.__new__(_cabi.NativeKernels)
    K.lib, K.launches = Lib(), 0
    monkeypatch.setattr(_cabi, "_on_device", lambda dev: __import__("contextlib").nullcontext())
    monkeypatch.setattr(K, "_stream", lambda t: 0, raising=False)
    a, b, c = z(4, 16), z(4, 24)[:, 8:], z(1, 8)
    assert all(x is y for x, y in zip(K.aligned_rows(a, b, c), (a, b, c))) and not calls
    out = K.aligned_rows(a, z(4, 9), z(3, 20)[:, 1:9], z(1, 8).expand(5, 8), z(1, 9))
    assert out[0] is a and calls == [[(4, 9, 9, 16), (3, 8, 20, 8), (5, 8, 0, 8)]]
    assert [tuple(t.shape) for t in out] == [(4, 16), (4, 9), (3, 8), (5, 8), (1, 9)] and K.launches == 1
    assert K.aligned_rows(z(8, 4).t())[0].is_contiguous()
