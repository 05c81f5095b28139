"""Derivatives that the training-step operators do not have are refused, not
lost: forward-mode tangents, and the gradient of a weight whose rows go to a
given output."""
import pytest
import torch
from torch.autograd import forward_ad

from suika_amd import (PlanError, clip_grads, grad_norm, grad_square_sum, token_logprobs, token_logprobs_grad,
                       vocab_embedding, vocab_embedding_grad)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("wants", [False, True])
def test_tangents_are_refused(wants):
    tokens, weight = torch.tensor([1, 2], device=DEV), torch.randn(4, 8, device=DEV)
    logits, targets = torch.randn(2, 5, device=DEV), torch.tensor([1, 2], device=DEV)
    one = torch.ones(2, device=DEV)
    r = token_logprobs(logits, targets)
    weight.requires_grad_(wants)
    logits.requires_grad_(wants)
    with forward_ad.dual_level():
        for call in (lambda: vocab_embedding(tokens, dual(weight)),
                     lambda: vocab_embedding_grad(tokens, dual(torch.ones(2, 8, device=DEV)), 4),
                     lambda: token_logprobs(dual(logits), targets),
                     lambda: token_logprobs_grad(dual(logits), targets, r.lse, r.entropy, one),
                     lambda: token_logprobs_grad(logits, targets, r.lse, r.entropy, dual(one)),
                     lambda: grad_norm([dual(one)]), lambda: grad_square_sum([dual(one)]),
                     lambda: clip_grads([dual(one)], 1.0)):
            with pytest.raises((PlanError, NotImplementedError, RuntimeError), match="forward|jvp"):
                call()
        # without tangents they work inside a level as well
        assert vocab_embedding(tokens, weight).shape == (2, 8)
        assert token_logprobs(logits, targets).logprob.shape == (2,)


def test_an_output_drops_no_gradient():
    tokens, out = torch.tensor([1, 2], device=DEV), torch.zeros(2, 8, device=DEV)
    weight = torch.randn(4, 8, device=DEV, requires_grad=True)
    with pytest.raises(PlanError, match="out"):
        vocab_embedding(tokens, weight, out=out)
    assert not bool(out.any())
    with torch.no_grad():
        vocab_embedding(tokens, weight, out=out)
    assert torch.equal(out, weight.detach()[tokens])
