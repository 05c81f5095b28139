"""Rows outside the shard, and gradients of rows without tokens, are zeros --
positive ones, in every column -- whatever the scale is."""
import math

import pytest
import torch

from suika_amd import vocab_embedding, vocab_embedding_grad

pytestmark = pytest.mark.gpu
DEV = "cuda"


def positive_zeros(t):
    return not bool(t.any()) and not bool(t.signbit().any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [3, 60, 257, 2053])
@pytest.mark.parametrize("scale", [2.0, -2.0, math.inf, -math.inf, math.nan])
def test_zero_rows(cols, scale, dtype):
    g = torch.Generator(DEV).manual_seed(1)
    weight = torch.rand(6, cols, generator=g, device=DEV).add_(0.5).to(dtype)
    tokens = torch.tensor([-1, 1, 6, 2 ** 40, 5], device=DEV)
    got = vocab_embedding(tokens, weight, scale=scale)
    assert positive_zeros(got[[0, 2, 3]])
    want = weight[[1, 5]].double() * scale
    assert torch.equal(got[[1, 4]].double().isnan(), want.isnan())
    assert torch.equal(got[[1, 4]].double().isinf(), want.isinf())
    grad = vocab_embedding_grad(tokens, torch.ones(5, cols, device=DEV, dtype=dtype), 6, scale=scale)
    assert positive_zeros(grad[[0, 2, 3, 4]])
    assert torch.equal(grad[[1, 5]].float(), torch.full((2, cols), scale, device=DEV)) or math.isnan(scale)
