"""The diagonal gated recurrence: ``gated_recurrence``, ``gated_recurrence_decode``, ``gated_recurrence_step``.

``h_t = exp(g_t) * h_{t-1} + w_t * v_t`` for every channel on its own, ``o_t = h_t``: the token mixer that stacks of recurrent
layers put beside gated delta layers. No counterpart in the reference; the conventions are those of ``gdn2_attention``: ``g`` is
the float32 natural-log decay (``<= 0``), ``w`` the write gate, the state float32, outputs in ``v.dtype``, ``cu_seqlens`` packs
sequences along the token axis of one batch entry, decoding updates the state in place. Unlike it, ``gated_recurrence`` has
a gradient. All arithmetic runs in the CUDA kernels behind :mod:`gdn2_tilelang_b200._cabi` (``csrc/recurrence.cu``), in float32.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _cabi

__all__ = ["gated_recurrence", "gated_recurrence_decode", "gated_recurrence_step"]


def _check_rows(v, g, w):
    if v.dim() < 3:
        raise ValueError(f"expected [B, S, ...] tensors, got shape {tuple(v.shape)}")
    if g.shape != v.shape or (w is not None and w.shape != v.shape):
        raise ValueError("v, g and w must share one shape")
    _cabi.dtype_code(v.dtype)
    if w is not None and w.dtype != v.dtype:
        raise TypeError("v and w must share one dtype")
    if not g.is_floating_point():
        raise TypeError(f"g must be a floating-point tensor, got {g.dtype}")
    _check_devices(v, g, w)


def _check_devices(v, *others):
    _cabi._require_cuda(v, *others)
    for t in others:
        if t is not None and t.device != v.device:
            raise ValueError(f"all tensors must be on one device, got {v.device} and {t.device}")


def _offsets(cu_seqlens, v):
    offs = [int(x) for x in (cu_seqlens.tolist() if torch.is_tensor(cu_seqlens) else cu_seqlens)]
    B, T = v.shape[:2]
    if B != 1:
        raise ValueError("with cu_seqlens the sequences are packed into one batch entry: expected B == 1")
    if len(offs) < 2 or offs[0] != 0 or offs[-1] != T or any(hi < lo for lo, hi in zip(offs, offs[1:])):
        raise ValueError(f"cu_seqlens must rise from 0 to the packed length {T}, got {offs}")
    return offs


class _GatedRecurrence(torch.autograd.Function):
    """``[B, S, D]`` rows, ``state [sequences, D]``; the forward pass leaves the states its backward pass starts from."""

    @staticmethod
    def forward(ctx, v, g, w, state, offsets):
        K = _cabi.kernels()
        o, final, marks = K.recurrence(v, g, w, state, offsets, want_marks=True)
        ctx.save_for_backward(v, g, w, marks)
        ctx.offsets, ctx.has_state = offsets, state is not None
        ctx.set_materialize_grads(False)
        return o, final

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dfinal):
        if do is None and dfinal is None:
            return None, None, None, None, None
        _cabi.refuse_tracing("gated_recurrence")
        _cabi.refuse_tangents("gated_recurrence", do, dfinal)
        v, g, w, marks = ctx.saved_tensors
        K = _cabi.kernels()
        do = torch.zeros_like(v) if do is None else do
        dv, dg, dw, dstate = K.recurrence_backward(v, g, w, marks, do, dfinal, ctx.offsets, ctx.has_state)
        K.maybe_check_device_status(v.device)
        return dv, dg, dw, dstate, None


def _plain(v, g, w, state, want_final, in_place=False, offsets=()):
    """The call in one native function, gradient included, where the extension takes it: ``(o, final_state | None)``, or ``None``.
    With a status check after every call, backward passes go through Python, too."""
    K = _cabi.kernels()
    call = getattr(getattr(K, "host", None), "recurrence", None)
    if call is None or K.checks_status:
        return None
    res = call(v, g, w, state, want_final, in_place, offsets)
    if res is None:
        return None
    K._launches += res[2]
    return res[0], res[1]


def gated_recurrence(v, g, w=None, initial_state=None, output_final_state=False, cu_seqlens=None):
    """``h_t = exp(g_t) * h_{t-1} + w_t * v_t`` along the tokens of whole sequences; differentiable in
    reverse mode, once.

    ``v, g, w``: ``[B, S, ...]``, one shape; all trailing dimensions are channels. ``v`` and ``w`` are float16, bfloat16 or
    float32, ``g`` (``<= 0``, ``-inf`` forgets the state) is coerced to float32; ``w=None`` writes ``v`` as it is.
    ``initial_state``: ``[B, ...]``, or zero. Returns ``(o [B, S, ...] in v.dtype, final_state [B, ...] float32 | None)``.

    Rows may be columns of a wider tensor (a fused projection): any batch and token stride is read in place as long as a
    token's channels lie side by side. Rows that start on 16 bytes and hold a multiple of 16 bytes take the fast kernels.

    ``cu_seqlens`` (``[N + 1]`` token offsets rising from 0 to ``S``, best on the host; ``B == 1``): ``N`` sequences packed along the
    token axis; ``initial_state`` and ``final_state`` are then ``[N, ...]``. An empty sequence hands its state through.

    A backward pass that is captured into a CUDA graph follows PyTorch's rule for it: no other graph of the same leaves alive
    on another stream (``torch.autograd.grad`` on inputs made for the capture is safe).
    """
    if g.dtype is not torch.float32 and g.is_floating_point():
        g = g.float()
    if initial_state is not None and initial_state.is_floating_point():
        initial_state = initial_state.float()
    if cu_seqlens is None and v.is_cuda:
        res = _plain(v, g, w, initial_state, output_final_state)
        if res is not None:
            return res
    _check_rows(v, g, w)
    _cabi.refuse_tracing("gated_recurrence")
    _cabi.refuse_tangents("gated_recurrence", v, g, w, initial_state)
    B, S = v.shape[:2]
    channels = tuple(v.shape[2:])
    offsets = None if cu_seqlens is None else _offsets(cu_seqlens, v)
    N = B if offsets is None else len(offsets) - 1
    if initial_state is not None:
        if tuple(initial_state.shape) != (N, *channels):
            raise ValueError(f"initial_state must have shape {(N, *channels)}, got {tuple(initial_state.shape)}")
        if not initial_state.is_floating_point():
            raise TypeError(f"initial_state must be a floating-point tensor, got {initial_state.dtype}")
        _check_devices(v, initial_state)
    if offsets is not None:
        res = _plain(v, g, w, initial_state, output_final_state, offsets=offsets)
        if res is not None:
            return res
    if v.numel() == 0:                                 # nothing to compute: the states pass through
        final = torch.zeros(N, *channels, dtype=torch.float32, device=v.device) if initial_state is None else initial_state.clone()
        o = torch.empty_like(v, memory_format=torch.contiguous_format)
        ins = [t for t in (v, g, w, initial_state) if t is not None and t.requires_grad]
        if torch.is_grad_enabled() and ins:            # zero gradients, from sums of no elements
            nothing = sum(t[:0].sum() for t in ins)
            o, final = o.detach() + nothing.to(o.dtype), final + nothing.float()
        return o, (final if output_final_state else None)
    rows = [None if t is None else t.flatten(2) for t in (v, g, w)]
    state = None if initial_state is None else initial_state.reshape(N, -1)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (v, g, w, initial_state)):
        o, final = _GatedRecurrence.apply(*rows, state, offsets)
    else:
        o, final, _ = _cabi.kernels().recurrence(*rows, state, offsets, want_final=output_final_state)
    _cabi.kernels().maybe_check_device_status(v.device)
    return o.view(v.shape), (final.view(N, *channels) if output_final_state else None)


def gated_recurrence_decode(v, g, w, state):
    """Decode ``n`` tokens (``[B, n, ...]``), updating ``state [B, ...]`` (float32, contiguous) in place. ``w`` may be ``None``.

    Returns ``o [B, n, ...]`` in ``v.dtype``. No gradient."""
    if g.dtype is not torch.float32 and g.is_floating_point():
        g = g.float()
    if v.is_cuda:
        res = _plain(v, g, w, state, True, in_place=True)
        if res is not None:
            return res[0]
    _check_rows(v, g, w)
    _cabi.refuse_tracing("gated_recurrence_decode")
    _cabi.refuse_tangents("gated_recurrence_decode", v, g, w, state)
    B = v.shape[0]
    if tuple(state.shape) != (B, *v.shape[2:]):
        raise ValueError(f"state must have shape {(B, *v.shape[2:])}, got {tuple(state.shape)}")
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError("the recurrent state must be a contiguous float32 tensor")
    _check_devices(v, state)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (v, g, w, state)):
        raise ValueError("decoding updates the state in place and has no gradient; call it under torch.no_grad() or detach the inputs")
    if v.numel() == 0:
        return torch.empty_like(v, memory_format=torch.contiguous_format)
    K = _cabi.kernels()
    rows = [None if t is None else t.flatten(2) for t in (v, g, w)]
    o, _, _ = K.recurrence(*rows, state.view(B, -1), None, in_place=True)
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)  # autograd sees that it was written
    K.maybe_check_device_status(v.device)
    return o.view(v.shape)


def gated_recurrence_step(v, g, w, state):
    """One token with ``[B, ...]``-shaped inputs; ``state`` is updated in place. Returns ``o [B, ...]``."""
    if v.dim() < 2:
        raise ValueError(f"expected [B, ...] tensors, got shape {tuple(v.shape)}")
    return gated_recurrence_decode(v.unsqueeze(1), g.unsqueeze(1), None if w is None else w.unsqueeze(1), state)[:, 0]
