"""The gated feed-forward block: ``gated_feed_forward`` and the ``GatedFeedForward`` module.

``y = (act(x Wg^T) * (x Wu^T)) Wd^T``: the channel mixer that follows every token mixer of a language model, beside the
``GatedDeltaNet2`` layer and the diagonal recurrence. No counterpart in the reference, which has the token mixer alone.
All arithmetic runs in the CUDA kernels behind :mod:`gdn2_tilelang_b200._cabi` (``csrc/ffn.cu``): both projections, the activation and
the product are one tensor-core kernel, the output projection another; a few tokens take kernels that read the weights once
across all SMs. float16 and bfloat16, sums in float32.
"""

from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _cabi

__all__ = ["gated_feed_forward", "GatedFeedForward"]


def _check(x, w_gate, w_up, w_down, activation):
    if activation not in _cabi.ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}; expected one of {tuple(_cabi.ACTIVATIONS)}")
    if any(w.dim() != 2 for w in (w_gate, w_up, w_down)) or x.dim() < 1:
        raise ValueError("expected x [..., hidden] and weights of two dimensions")
    inner, hidden = w_gate.shape
    if w_up.shape != w_gate.shape or w_down.shape[1] != inner or x.shape[-1] != hidden:
        raise ValueError("expected x [..., hidden], w_gate and w_up [inner, hidden], w_down [out, inner], got "
                         f"{tuple(x.shape)}, {tuple(w_gate.shape)}, {tuple(w_up.shape)}, {tuple(w_down.shape)}")
    if hidden == 0 or inner == 0 or w_down.shape[0] == 0:
        raise ValueError("hidden, inner and output sizes must be positive")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"unsupported dtype {x.dtype}; use float16 or bfloat16 (float32 weights: under torch.autocast)")
    if any(w.dtype != x.dtype for w in (w_gate, w_up, w_down)):
        raise TypeError("x and the weights must share one dtype")
    _cabi._require_cuda(x, w_gate, w_up, w_down)
    if any(w.device != x.device for w in (w_gate, w_up, w_down)):
        raise ValueError("x and the weights must be on one device")


class _GatedFeedForward(torch.autograd.Function):
    """``x [tokens, hidden]``, at least one token."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        K = _cabi.kernels()
        ins = K.aligned_rows(x, w_gate, w_up, w_down)
        y, kept = K.ffn_forward(*ins, activation, keep=True)
        ctx.save_for_backward(*ins, kept)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        K = _cabi.kernels()
        _cabi.refuse_tracing("gated_feed_forward")
        _cabi.refuse_tangents("gated_feed_forward", dy)
        need = ctx.needs_input_grad
        dx, dwg, dwu, dwd = K.ffn_backward(*ctx.saved_tensors, dy, ctx.activation, need[0], need[1] or need[2], need[3])
        K.maybe_check_device_status(dy.device)
        return dx, (dwg if need[1] else None), (dwu if need[2] else None), dwd, None


def _autocast(*tensors):
    """What ``nn.Linear`` would do inside an autocast region: operands of up to 32 bits in the region's type."""
    to = torch.get_autocast_dtype("cuda")
    return tuple(t.to(to) if t.is_cuda and t.dtype in (torch.float32, torch.float16, torch.bfloat16) else t for t in tensors)


def gated_feed_forward(x, w_gate, w_up, w_down, activation="silu"):
    """``(act(x w_gate^T) * (x w_up^T)) w_down^T``; differentiable in reverse mode, once.

    ``x``: ``[..., hidden]``; ``w_gate, w_up``: ``[inner, hidden]``; ``w_down``: ``[out, inner]`` (the layout of ``nn.Linear``), all float16
    or all bfloat16; inside ``torch.autocast`` they are cast to its type first, so float32 weights train there. ``activation``: ``"silu"`` or ``"gelu_tanh"``. Returns ``[..., out]``. What one product
    reads of another is rounded to the inputs' type, sums are float32; a graph keeps 6 bytes an inner channel and token.

    Any sizes and row strides. Rows that do not start on 16 bytes (a size that is not a multiple of 8, an odd slice) are copied
    first, in one launch for all operands.
    """
    if torch.is_autocast_enabled("cuda"):
        x, w_gate, w_up, w_down = _autocast(x, w_gate, w_up, w_down)
    if x.is_cuda and activation in _cabi.ACTIVATIONS:
        K = _cabi.kernels()
        call = getattr(getattr(K, "host", None), "feed_forward", None)
        if call is not None and not K.checks_status:       # the call in one native function, gradient included
            res = call(x, w_gate, w_up, w_down, _cabi.ACTIVATIONS[activation])
            if res is not None:
                K._launches += res[1]
                return res[0]
    _check(x, w_gate, w_up, w_down, activation)
    _cabi.refuse_tracing("gated_feed_forward")
    _cabi.refuse_tangents("gated_feed_forward", x, w_gate, w_up, w_down)
    out_shape = (*x.shape[:-1], w_down.shape[0])
    needs_grad = torch.is_grad_enabled() and any(t.requires_grad for t in (x, w_gate, w_up, w_down))
    if x.numel() == 0:                                 # no tokens: an empty result, zero gradients
        y = x.new_empty(out_shape)
        return y + sum(t.sum() * 0 for t in (x, w_gate, w_up, w_down)) if needs_grad else y
    rows = x.reshape(-1, x.shape[-1])
    if needs_grad:
        y = _GatedFeedForward.apply(rows, w_gate, w_up, w_down, activation)
    else:
        K = _cabi.kernels()
        y = K.ffn_forward(*K.aligned_rows(rows, w_gate, w_up, w_down), activation, keep=False)[0]
    _cabi.kernels().maybe_check_device_status(x.device)
    return y.view(out_shape)


class GatedFeedForward(nn.Module):
    """``gated_feed_forward`` with its weights: ``gate_proj``, ``up_proj`` (``hidden -> intermediate``) and ``down_proj``
    (``intermediate -> hidden``), ``nn.Linear`` modules without biases that hold the parameters. They are made in the default type:
    convert the module to float16 or bfloat16, or call it inside ``torch.autocast``."""

    def __init__(self, hidden_size: int, intermediate_size: int, activation: str = "silu"):
        super().__init__()
        if activation not in _cabi.ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}; expected one of {tuple(_cabi.ACTIVATIONS)}")
        self.hidden_size, self.intermediate_size, self.activation = hidden_size, intermediate_size, activation
        self.gate_proj = nn.Linear(hidden_size, intermediate_size, bias=False)
        self.up_proj = nn.Linear(hidden_size, intermediate_size, bias=False)
        self.down_proj = nn.Linear(intermediate_size, hidden_size, bias=False)

    def forward(self, x):
        return gated_feed_forward(x, self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight, self.activation)

    def extra_repr(self):
        return f"activation={self.activation!r}"
