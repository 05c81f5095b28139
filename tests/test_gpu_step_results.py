"""The gradient of the logits has their type, and an output that is given is
what comes back."""
import pytest
import torch

from suika_amd import token_logprobs, token_logprobs_grad, vocab_embedding

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_gradient_has_the_logits_type(dtype):
    g = torch.Generator(DEV).manual_seed(1)
    logits = torch.randn(3, 10, generator=g, device=DEV).to(dtype)
    targets, one = torch.tensor([1, 2, 3], device=DEV), torch.ones(3, device=DEV)
    r = token_logprobs(logits, targets)
    assert token_logprobs_grad(logits, targets, r.lse, r.entropy, one, one).dtype == dtype
    out = torch.empty_like(logits)
    got = token_logprobs_grad(logits, targets, r.lse, r.entropy, one, one, out=out)
    assert got.data_ptr() == out.data_ptr() and got.dtype == dtype


def test_a_given_output_is_what_comes_back():
    g = torch.Generator(DEV).manual_seed(2)
    weight, tokens = torch.randn(8, 16, generator=g, device=DEV), torch.tensor([1, 9, 3], device=DEV)
    want = vocab_embedding(tokens, weight)
    out = torch.full((3, 16), 7.0, device=DEV)
    got = vocab_embedding(tokens, weight, out=out)
    assert got.data_ptr() == out.data_ptr() and got.shape == out.shape
    assert torch.equal(out, want) and torch.equal(got, want)
