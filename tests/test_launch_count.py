"""Counting launches costs a call an addition: gradients' launches, which the host extension counts, are asked for where the count is
read. No GPU."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from gdn2_tilelang_b200 import _cabi


class Host:
    asked = 0

    def gradient_launches(self):
        Host.asked += 1
        return 5

    def decode(self, q, k, v, g, b, w, state, scale):
        return torch.zeros_like(v)

    def prefill_short(self, q, k, v, g, b, w, scale, state):
        return torch.zeros_like(v), torch.zeros(1, 2, 8, 8)

    def recurrence(self, v, g, w, state, want_final, in_place, offsets):
        return torch.zeros_like(v), state, 1


@pytest.fixture
def K(monkeypatch):
    k = _cabi.NativeKernels.__new__(_cabi.NativeKernels)
    k.lib, k.host, k.launches, Host.asked = None, Host(), 0, 0
    monkeypatch.setattr(_cabi, "_kernels", k)
    monkeypatch.delenv("GDN2_B200_CHECK_STATUS", raising=False)
    Host.asked = 0
    return k


def test_calls_do_not_ask_for_the_gradients_count(K):
    x, step, state = torch.zeros(1, 3, 2, 8), torch.zeros(1, 2, 8), torch.zeros(1, 2, 8, 8)
    gdn2.gdn2_decode(*[x] * 6, state)
    gdn2.gdn2_decode_step(*[step] * 6, state)
    gdn2.gdn2_prefill(*[x] * 6)
    assert Host.asked == 0
    assert K.launches == 3 and Host.asked == 1             # set to 0 when five gradients had been counted, which are not new


def test_the_count_holds_what_gradients_launched(K, monkeypatch):
    before = K.launches
    monkeypatch.setattr(Host, "gradient_launches", lambda self: 7)
    assert K.launches == before + 2
    K.launches = 11
    assert K.launches == 11
    del K.host
    k = _cabi.NativeKernels.__new__(_cabi.NativeKernels)
    k.launches = 4                                          # before there is an extension
    assert k.launches == 4
