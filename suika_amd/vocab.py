"""The vocabulary's ends of a model: the embedding of a shard, and what the
head's logits say about given tokens.

* ``vocab_embedding``       -- rows of a vocabulary shard for given tokens;
* ``vocab_embedding_grad``  -- the gradient of those rows;
* ``token_logprobs``        -- log probabilities of given tokens, entropy and
                               the best alternatives;
* ``token_logprobs_grad``   -- the gradient of the logits.

A rank holds the rows ``vocab_start .. vocab_start + len(weight)`` of the
embedding (the ``vocab_pad`` shards of a ``ParamLayout``; the whole table at
tensor-parallel degree 1, as the reference's nn.Embedding,
Suika/models/llama_model.py:108-157).  Tokens of other ranks give zeros and no
gradient, so the ranks' outputs add up to the embedding.  The head's logits
are whole, as the reference gathers them (lm_head is column parallel with
``gather_output``, Suika/tensor_parallel.py:486-606); where its rows are
padded, ``vocab`` says how many are tokens.

The kernels run on the tensors' device, on its current stream, behind the C
ABI of include/suika_step.h.  Refused arguments raise ``PlanError``, and so do
forward-mode tangents, which the operators do not have.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import _lib
from ._lib import PlanError


def vocab_embedding(tokens: Tensor, weight: Tensor, *, scale: float = 1.0, vocab_start: int = 0,
                    out: Optional[Tensor] = None) -> Tensor:
    """``scale * weight[tokens - vocab_start]``, zeros for tokens outside the
    shard (negative ones among them); of shape ``tokens.shape + (columns,)``.

    ``tokens`` are int64 or int32 and contiguous, ``weight`` is float32,
    bfloat16 or float16 with dense rows at any distance.  Products are rounded
    once.  Where ``weight`` wants a gradient, the result is differentiable
    (``vocab_embedding_grad``, in the weight's type), and ``out`` is refused.
    """
    if weight.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise PlanError("out: the weight wants a gradient, which rows in a given output do not have")
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


class _Results(NamedTuple):
    logprob: Tensor
    entropy: Tensor
    lse: Tensor
    top_logprob: Optional[Tensor]
    top_index: Optional[Tensor]


class TokenLogprobs(_Results):
    """What ``token_logprobs`` returns: float32 tensors of the targets' shape,
    and the alternatives (with one more dimension) or ``None``.

    ``lse_low``, which is not one of the tuple's items, is what the rounding
    of ``lse`` to float32 lost: ``token_logprobs_grad`` takes both where the
    logits have a large common offset.
    """
    lse_low: Optional[Tensor] = None

    @classmethod
    def _of(cls, results) -> "TokenLogprobs":
        r = cls(*results[:5])
        r.lse_low = results[5]
        return r


def token_logprobs(logits: Tensor, targets: Tensor, *, top: int = 0, vocab: Optional[int] = None) -> TokenLogprobs:
    """Log probabilities of ``targets`` under ``logits``, with the entropy and
    the ``lse`` (log of the sum of the exponentials) of each row.

    ``logits`` are float32, bfloat16 or float16 with dense rows, all one
    distance apart (``logits[..., :n]`` of a contiguous tensor, for example);
    their first ``vocab`` columns (default: all) are tokens.  ``targets``
    (int64 or int32) has the other dimensions.  A negative target, as
    ``ignore_index=-100``, is not scored: logprob 0.  A target of ``vocab``
    or more has logprob -inf.  ``top`` (at most 64) asks for the largest log
    probabilities in falling order, int64 columns with them; equal logits come
    by column.  Statistics are formed in 32 bits.

    A row whose logits are all -inf has lse and logprobs -inf and entropy 0;
    a row with NaN or +inf has NaN statistics, and its alternatives have NaN
    above +inf.

    Where ``logits`` want a gradient, ``logprob`` and ``entropy`` are
    differentiable (``token_logprobs_grad``); ``lse`` and the alternatives are
    not.
    """
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs._of(_Logprobs.apply(logits, targets, top, vocab))
    return TokenLogprobs._of(_lib.host().token_logprobs(logits, targets, top, vocab))


def token_logprobs_grad(logits: Tensor, targets: Tensor, lse: Tensor, entropy: Tensor,
                        grad_logprob: Optional[Tensor], grad_entropy: Optional[Tensor] = None, *,
                        vocab: Optional[int] = None, out: Optional[Tensor] = None,
                        lse_low: Optional[Tensor] = None) -> Tensor:
    """The gradient of the logits from those of ``logprob`` and ``entropy``
    (float32 of the targets' shape, or ``None``), in the logits' type:
    ``grad_logprob ([j = target] - p_j) - grad_entropy p_j (ln p_j + entropy)``.

    ``lse`` and ``entropy`` are what ``token_logprobs`` returned, and so is
    ``lse_low``; without it, p_j is off by up to ``|lse| 2^-24`` of itself, as
    ``lse`` is rounded to float32.  Padded columns and rows that are all -inf
    get 0, and a row that is not scored has no first term.  ``out`` may be
    ``logits`` itself.
    """
    return _lib.host().token_logprobs_grad(logits, targets, lse, entropy, grad_logprob, grad_entropy, vocab, out,
                                           lse_low)


class _Logprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, vocab):
        r = _lib.host().token_logprobs(logits, targets, top, vocab)
        ctx.save_for_backward(logits, targets, r[2], r[1], r[5])
        ctx.vocab = vocab
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*[t for t in r[2:] if t is not None])
        return r

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logprob, grad_entropy, *others):
        if grad_logprob is None and grad_entropy is None:
            return None, None, None, None
        logits, targets, lse, entropy, lse_low = ctx.saved_tensors
        grads = [None if g is None else g.contiguous() for g in (grad_logprob, grad_entropy)]
        grad = token_logprobs_grad(logits, targets, lse, entropy, *grads, vocab=ctx.vocab, lse_low=lse_low)
        return grad, None, None, None
