"""The training-step operators on tensors whose storage was released, as
forcefully_free_tensor does it with a source: at offset 0 such a tensor's
address is null, as a view into a larger allocation its offset alone.  Every
call refuses it on the host, before anything runs."""
import pytest
import torch

from suika_amd import (PlanError, ShardAdamW, clip_grads, forcefully_free_tensor, grad_norm, grad_square_sum,
                       token_logprobs, token_logprobs_grad, vocab_embedding, vocab_embedding_grad)

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def released(shape, dtype=F32, offset=0, cols=None):
    """A tensor of an allocation of its own, ``offset`` elements into it, and
    released; with ``cols``, its first columns."""
    n = torch.Size(shape).numel()
    t = torch.zeros(n + offset, dtype=dtype, device=DEV)[offset:].view(shape)
    if cols is not None:
        t = t[:, :cols]
    forcefully_free_tensor(t)
    assert t.untyped_storage().nbytes() == 0 and t.numel() > 0
    return t


def state_of(n=64):
    w = torch.arange(n, device=DEV, dtype=F32)
    return {"w": {"param": w.to(BF16), "master": w, "exp_avg": torch.ones(n, device=DEV),
                  "exp_avg_sq": torch.ones(n, device=DEV), "step": torch.tensor(3.0)}}


@pytest.mark.parametrize("offset", [0, 64])
@pytest.mark.parametrize("field", ["param", "master", "exp_avg", "exp_avg_sq"])
def test_step_refuses_a_released_field(field, offset):
    state = state_of()
    whole = torch.zeros(64 + offset, dtype=state["w"][field].dtype, device=DEV)
    whole[offset:] = state["w"][field]
    state["w"][field] = whole[offset:]
    opt = ShardAdamW(state)
    before = {f: t.clone() for f, t in state["w"].items()}
    versions = {f: t._version for f, t in state["w"].items()}
    forcefully_free_tensor(whole)
    with pytest.raises(PlanError, match="w: a field's storage has been released"):
        opt.step([torch.ones(64, device=DEV)], max_norm=1.0)
    torch.cuda.synchronize()
    for f, t in state["w"].items():
        assert t._version == versions[f]
        assert f == field or torch.equal(t, before[f])
    assert opt.steps == 3
    with pytest.raises(PlanError, match="released"):
        ShardAdamW(state)


@pytest.mark.parametrize("offset", [0, 64])
def test_gradients(offset):
    grads = [torch.ones(8, device=DEV), released((64,), F32, offset)]
    opt = ShardAdamW(state_of())
    out = [torch.zeros(8, device=DEV), torch.zeros(64, device=DEV)]
    for call in (lambda: grad_norm(grads), lambda: grad_square_sum(grads), lambda: clip_grads(grads, 1.0),
                 lambda: clip_grads(grads, 1.0, out=out), lambda: clip_grads(out, 1.0, out=grads),
                 lambda: opt.step(grads[1:]), lambda: opt.step(out[1:], max_norm=1.0, square_sum=released((), torch.float64, offset)),
                 lambda: clip_grads(out, 1.0, square_sum=released((), torch.float64, offset))):
        with pytest.raises(PlanError, match="released"):
            call()
    assert opt.steps == 3 and not bool(out[0].any()) and bool((grads[0] == 1).all())


@pytest.mark.parametrize("offset", [0, 64])
def test_embedding(offset):
    tokens, weight = torch.zeros(4, dtype=torch.int64, device=DEV), torch.zeros(8, 16, device=DEV)
    grad = torch.zeros(4, 16, device=DEV)
    for call in (lambda: vocab_embedding(released((4,), torch.int64, offset), weight),
                 lambda: vocab_embedding(tokens, released((8, 16), F32, offset)),
                 lambda: vocab_embedding(tokens, released((8, 32), F32, offset, cols=16)),
                 lambda: vocab_embedding(tokens, weight, out=released((4, 16), F32, offset)),
                 lambda: vocab_embedding_grad(released((4,), torch.int64, offset), grad, 8),
                 lambda: vocab_embedding_grad(tokens, released((4, 16), F32, offset), 8),
                 lambda: vocab_embedding_grad(tokens, grad, 8, out=released((8, 16), F32, offset))):
        with pytest.raises(PlanError, match="released"):
            call()
    assert vocab_embedding(tokens[:0], weight).shape == (0, 16)


@pytest.mark.parametrize("offset", [0, 64])
def test_log_probabilities(offset):
    logits, targets = torch.zeros(4, 16, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    r = token_logprobs(logits, targets)
    one, gone = torch.ones(4, device=DEV), released((4,), F32, offset)
    for call in (lambda: token_logprobs(released((4, 16), F32, offset), targets),
                 lambda: token_logprobs(logits, released((4,), torch.int64, offset)),
                 lambda: token_logprobs_grad(released((4, 16), F32, offset), targets, r.lse, r.entropy, one),
                 lambda: token_logprobs_grad(logits, released((4,), torch.int64, offset), r.lse, r.entropy, one),
                 lambda: token_logprobs_grad(logits, targets, gone, r.entropy, one),
                 lambda: token_logprobs_grad(logits, targets, r.lse, gone, one),
                 lambda: token_logprobs_grad(logits, targets, r.lse, r.entropy, gone),
                 lambda: token_logprobs_grad(logits, targets, r.lse, r.entropy, None, gone),
                 lambda: token_logprobs_grad(logits, targets, r.lse, r.entropy, one, out=released((4, 16), F32, offset))):
        with pytest.raises(PlanError, match="released"):
            call()
