"""The gated feed-forward block of a tensor-parallel share.

* ``gated_ffn``       -- ``act(x gate^T) * (x up^T)`` times ``down^T``;
* ``gated_ffn_grad``  -- the gradients of the input and the three matrices.

A rank holds rows of ``gate`` and ``up`` (column parallel) and the same columns
of ``down`` (row parallel), as the reference's Llama and Qwen2 blocks do
(Suika/models/llama_model.py:16-35, Suika/models/qwen_model.py:17-40), so the
ranks' outputs, and their gradients of ``x``, add up.  The matrices are the
``mlp`` entries of a state that ``execute_param_transfer`` returns.

The kernels run on the tensors' device, on its current stream, behind the C
ABI of include/suika_step.h.  Refused arguments raise ``PlanError``, and so do
forward-mode tangents, which the operators do not have.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from ._lib import PlanError


class GatedFFN(NamedTuple):
    """What ``gated_ffn`` returns with ``keep``: its output, and the two
    projections, ``x gate^T`` and ``x up^T`` in float32, that
    ``gated_ffn_grad`` takes."""
    out: Tensor
    gate: Tensor
    up: Tensor


def gated_ffn(x: Tensor, gate: Tensor, up: Tensor, down: Tensor, *, activation: str = "silu",
              keep: bool = False) -> Union[Tensor, GatedFFN]:
    """``(act(x gate^T) * (x up^T)) down^T``, of ``x``'s shape.

    ``x`` is ``[..., hidden]``, ``gate`` and ``up`` are ``[ffn, hidden]`` and
    ``down`` is ``[hidden, ffn]``, all float32, bfloat16 or float16 with dense
    rows one distance apart; any size may be 0.  ``activation`` is ``"silu"``,
    ``"gelu"`` or ``"gelu_tanh"``.  Sums are formed in 32 bits; the product of
    the activation and the second projection is rounded to the tensors' type
    before the last product, and in float16 has to lie in its range.

    Where a tensor wants a gradient, the result is differentiable in all four.
    ``keep`` asks for the projections, for a ``gated_ffn_grad`` by hand; they
    are not differentiable.
    """
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, gate, up, down)):
        if keep:
            raise PlanError("keep: a tensor wants a gradient, which autograd then forms by itself")
        return _GatedFFN.apply(x, gate, up, down, activation)
    r = _lib.host().gated_ffn(x, gate, up, down, activation, keep)
    return GatedFFN(*r) if keep else r[0]


def gated_ffn_grad(x: Tensor, gate: Tensor, up: Tensor, down: Tensor, kept_gate: Tensor, kept_up: Tensor,
                   grad_output: Tensor, *, activation: str = "silu",
                   wanted: Sequence[bool] = (True, True, True, True)) -> Tuple[Optional[Tensor], ...]:
    """The gradients of ``x``, ``gate``, ``up`` and ``down`` from that of the
    output, each in the tensors' type, or ``None`` where ``wanted`` says so.

    ``kept_gate`` and ``kept_up`` are what ``gated_ffn(..., keep=True)``
    returned of the same arguments.  Sums are formed in 32 bits; the gradients
    of the two projections are rounded to the tensors' type on the way.
    """
    return _lib.host().gated_ffn_grad(x, gate, up, down, kept_gate, kept_up, grad_output, activation, list(wanted))


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, up, down, activation):
        out, kept_gate, kept_up = _lib.host().gated_ffn(x, gate, up, down, activation, True)
        ctx.save_for_backward(x, gate, up, down, kept_gate, kept_up)
        ctx.activation = activation
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        grads = gated_ffn_grad(*ctx.saved_tensors, grad_output.contiguous(), activation=ctx.activation,
                               wanted=ctx.needs_input_grad[:4])
        return (*grads, None)
