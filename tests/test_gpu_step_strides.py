"""Rows of dense elements that are one distance apart are taken in tensors of
any number of dimensions; other strides are refused."""
import pytest
import torch

from suika_amd import PlanError, token_logprobs, token_logprobs_grad, vocab_embedding_grad

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


@pytest.mark.parametrize("lead", [(5, 6), (2, 3, 5), (1, 7), (7, 1), (2, 1, 4), (1, 1), (3, 1, 1, 2)])
def test_rows_of_more_dimensions(lead):
    g = gen(1)
    wide = torch.randn(*lead, 40, generator=g, device=DEV)
    targets = torch.randint(0, 30, lead, generator=g, device=DEV)
    one = torch.randn(lead, generator=g, device=DEV)
    for part in (wide[..., :30], wide[..., 7:37], wide[..., 3:4]):
        cols = part.shape[-1]
        whole = part.contiguous()
        t = targets.clamp(max=cols - 1)
        r, want = token_logprobs(part, t, top=1), token_logprobs(whole, t, top=1)
        assert all(torch.equal(a, b) for a, b in zip(r, want))
        grad = token_logprobs_grad(whole, t, r.lse, r.entropy, one, one)
        assert torch.equal(token_logprobs_grad(part, t, r.lse, r.entropy, one, one), grad)
        room = torch.full((*lead, 50), 5.0, device=DEV)
        into = room[..., 9:9 + cols]
        assert token_logprobs_grad(part, t, r.lse, r.entropy, one, one, out=into).data_ptr() == into.data_ptr()
        assert torch.equal(into, grad) and bool((room[..., :9] == 5).all()) and bool((room[..., 9 + cols:] == 5).all())
        tokens = targets % 4
        assert torch.equal(vocab_embedding_grad(tokens, part, 4), vocab_embedding_grad(tokens, whole, 4))


def test_other_strides_are_refused():
    g = gen(2)
    x = torch.randn(4, 6, 10, generator=g, device=DEV)
    t = torch.zeros(4, 6, dtype=torch.int64, device=DEV)
    for bad, targets in [(x[:, 1:], t[:, 1:].contiguous()), (x[:, ::2][:, :2], t[:, :2].contiguous()),
                         (x.transpose(0, 1), t.t().contiguous()), (x[..., ::2], t),
                         (x[:1].expand(4, 6, 10), t), (x[:, :1].expand(4, 6, 10), t),
                         (x.as_strided((4, 6, 10), (30, 5, 1)), t)]:
        with pytest.raises(PlanError, match="dense elements"):
            token_logprobs(bad, targets)
        with pytest.raises(PlanError, match="dense elements"):
            vocab_embedding_grad(targets, bad, 4)
    assert token_logprobs(x[::2, :1], t[::2, :1].contiguous()).lse.shape == (2, 1)      # every 12th row
