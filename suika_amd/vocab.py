"""The vocabulary's end of a training step: the embedding of a shard.

* ``vocab_embedding``       -- rows of a vocabulary shard for given tokens;
* ``vocab_embedding_grad``  -- the gradient of those rows.

A rank holds the rows ``vocab_start .. vocab_start + len(weight)`` of the
embedding (the ``vocab_pad`` shards of a ``ParamLayout``; the whole table at
tensor-parallel degree 1, as the reference's nn.Embedding,
Suika/models/llama_model.py:108-157).  Tokens of other ranks give zeros and no
gradient, so the ranks' outputs add up to the embedding.

The kernels run on the tensors' device, on its current stream, behind the C
ABI of include/suika_step.h.  Refused arguments raise ``PlanError``.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import _lib


def vocab_embedding(tokens: Tensor, weight: Tensor, *, scale: float = 1.0, vocab_start: int = 0,
                    out: Optional[Tensor] = None) -> Tensor:
    """``scale * weight[tokens - vocab_start]``, zeros for tokens outside the
    shard (negative ones among them); of shape ``tokens.shape + (columns,)``.

    ``tokens`` are int64 or int32 and contiguous, ``weight`` is float32,
    bfloat16 or float16 with dense rows at any distance.  Products are rounded
    once.  Where ``weight`` wants a gradient, the result is differentiable
    (``vocab_embedding_grad``, in the weight's type); ``out`` is for calls
    without.
    """
    if out is None and weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(tokens, weight, float(scale), int(vocab_start))
    return _lib.host().vocab_embedding(tokens, weight, scale, vocab_start, out)


def vocab_embedding_grad(tokens: Tensor, grad_output: Tensor, rows: int, *, scale: float = 1.0, vocab_start: int = 0,
                         dtype: Optional[torch.dtype] = None, out: Optional[Tensor] = None,
                         accumulate: bool = False) -> Tensor:
    """The gradient of a shard of ``rows`` rows: ``scale`` times the sum of
    ``grad_output`` over each row's tokens, zeros for rows without.

    The tokens are sorted and every row's are added in their order, in 32
    bits, so the result does not change from run to run.  It is of ``dtype``
    (default: that of ``grad_output``), or goes to ``out``, with
    ``accumulate`` on top of what is there (rows without tokens are not
    touched then).
    """
    return _lib.host().vocab_embedding_grad(tokens, grad_output, rows, scale, vocab_start, dtype, out, accumulate)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, vocab_start):
        ctx.save_for_backward(tokens)
        ctx.rows, ctx.dtype, ctx.scale, ctx.vocab_start = weight.shape[0], weight.dtype, scale, vocab_start
        return _lib.host().vocab_embedding(tokens, weight, scale, vocab_start, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        grad = vocab_embedding_grad(ctx.saved_tensors[0], grad_output.contiguous(), ctx.rows, scale=ctx.scale,
                                    vocab_start=ctx.vocab_start, dtype=ctx.dtype)
        return None, grad, None, None
