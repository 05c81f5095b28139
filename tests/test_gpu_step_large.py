"""The training-step operators beyond 2^31 elements and 2^32 bytes: the parts
that lie there are compared with the same rows or elements on their own."""
import pytest
import torch

from suika_amd import (ShardAdamW, clip_grads, grad_square_sum, token_logprobs, token_logprobs_grad, vocab_embedding,
                       vocab_embedding_grad)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def test_embedding_beyond_32_bits():
    rows, cols = 600_000, 4096                       # 2.5 G elements
    g = gen(1)
    weight = torch.empty(rows, cols, device=DEV, dtype=BF16).normal_(generator=g)
    tokens = torch.randint(0, rows, (3000,), generator=g, device=DEV)
    tokens[:400] = rows - 1
    assert torch.equal(vocab_embedding(tokens, weight), weight[tokens])
    grad_out = weight[:3000]
    grad = vocab_embedding_grad(tokens, grad_out, rows)
    hit, inverse = tokens.unique(return_inverse=True)
    small = vocab_embedding_grad(inverse, grad_out, len(hit))
    assert torch.equal(grad[hit], small)
    grad[hit] = 0
    assert not bool(grad.any())
    # outputs' gradients that lie beyond 32 bits
    far = torch.arange(rows, device=DEV) % 5
    sums = vocab_embedding_grad(far, weight, 5, dtype=torch.float32)
    want = torch.stack([weight[k::5].sum(0, dtype=torch.float64) for k in range(5)])
    size = torch.stack([weight[k::5].abs().sum(0, dtype=torch.float64) for k in range(5)])
    assert bool(((sums.double() - want).abs() <= rows / 5 * 2.0 ** -24 * size).all())


def test_logprobs_beyond_32_bits():
    rows, vocab = 16_000, 152_064                    # 2.4 G elements
    g = gen(2)
    logits = torch.empty(rows, vocab, device=DEV, dtype=BF16).normal_(generator=g)
    targets = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    one = torch.ones(rows, device=DEV)
    r = token_logprobs(logits, targets, top=3)
    tail = slice(rows - 70, rows)
    alone = logits[tail].clone()
    x = alone.double()
    lse = torch.logsumexp(x, 1)
    # a lane adds vocab / 256 exponentials; the bound is that of the small sizes
    bound = (vocab / 256 + 64) * 2.0 ** -24 + 8 * 2.0 ** -24 * lse.abs()
    assert bool(((r.lse[tail].double() - lse).abs() <= bound).all())
    chosen = x.gather(1, targets[tail][:, None])[:, 0] - lse
    assert bool(((r.logprob[tail].double() - chosen).abs() <= 2 * bound).all())
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :3]
    assert torch.equal(r.top_index[tail], order)
    grad = token_logprobs_grad(logits, targets, r.lse, r.entropy, one, one, out=logits)
    small = token_logprobs_grad(alone, targets[tail], r.lse[tail], r.entropy[tail], one[tail], one[tail])
    assert torch.equal(grad[tail], small)


def test_optimizer_beyond_32_bits():
    n = 2 ** 31 + 4099
    g = gen(3)
    state = {"w": {f: torch.empty(n, device=DEV).normal_(generator=g) for f in ("param", "exp_avg")}}
    state["w"]["exp_avg_sq"] = torch.empty(n, device=DEV).uniform_(generator=g)
    grad = torch.empty(n, device=DEV, dtype=BF16).normal_(generator=g)
    parts = [slice(0, 3000), slice(n - 6000, n)]
    small = [{"w": {f: t[p].clone() for f, t in state["w"].items()}} for p in parts]
    q = grad_square_sum([grad])
    want = sum(float(x.double().square().sum()) for x in grad.split(1 << 28))
    assert abs(float(q) - want) <= 1e-12 * want
    ShardAdamW(state).step([grad], max_norm=1.0)
    for p, s in zip(parts, small):
        ShardAdamW(s).step([grad[p].clone()], max_norm=1.0, square_sum=q)
        assert all(torch.equal(state["w"][f][p], s["w"][f]) for f in s["w"])
    clipped = grad.clone()
    clip_grads([clipped], 1.0, square_sum=q)
    for p in parts:
        one = grad[p].clone()
        clip_grads([one], 1.0, square_sum=q)
        assert torch.equal(clipped[p], one)
