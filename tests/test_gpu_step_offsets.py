"""The gradient of the logits where these have a large common offset, or are
all of the lowest value: with lse as a pair of floats, and through autograd,
the probabilities do not depend on the offset.

u = 2^-24.  The log of the sum is known to S = (V/256 + 64) u, as for the log
probabilities (a lane adds up to V/256 exponentials of a few u, the lanes are
joined in 8 steps).  x - lse is exact or off by u of itself, and its product
with log2 e by 2u, so p_j is known to S + 4u (|ln p_j| + 1) of itself whatever
lse is; the entropy, a mean of at most 2 ln V + 1, to S (2 + 3 ln V).  The sum of
a row's gradients is 0 but for their own errors."""
import math

import pytest
import torch

from suika_amd import TokenLogprobs, token_logprobs, token_logprobs_grad

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {t: torch.finfo(t).eps / 2 for t in (F32, BF16, F16)}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -25}
u = U[F32]
DEV = "cuda"


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def grad64(logits, targets, gl, gh, vocab):
    """(gradient, how far it may be off before it is rounded)"""
    x = logits[:, :vocab].double()
    x = x - x.amax(1, keepdim=True)
    logp = x - x.exp().sum(1, keepdim=True).log()
    p = logp.exp()
    ln_p = torch.where(p > 0, logp, 0.0)
    entropy = -(p * ln_p).sum(1, keepdim=True)
    gl = torch.where(targets >= 0, gl.double(), 0.0)[:, None]
    gh = gh.double()[:, None]
    hit = (torch.arange(vocab, device=DEV)[None] == targets[:, None]).double()
    grad = gl * (hit - p) - gh * p * (ln_p + entropy)
    S = (vocab / 256 + 64) * u
    known = S + 4 * u * (ln_p.abs() + 1)
    off = p * (gl.abs() + gh.abs() * (ln_p.abs() + entropy + 1)) * known
    off = off + p * gh.abs() * S * (2 + 3 * math.log(max(vocab, 2))) + 4 * u * gl.abs() * hit
    pad = (0, logits.shape[1] - vocab)
    return torch.nn.functional.pad(grad, pad), torch.nn.functional.pad(off, pad)


def near(got, want, off):
    allowed = off + U[got.dtype] * (want.abs() + off) + TINY[got.dtype]
    diff = (got.double() - want).abs()
    assert bool((diff <= allowed).all()), (float(diff.max()), float((diff / allowed).max()))
    # a row's sum, where all its gradients are formed from the same probabilities
    assert bool((got.double().sum(1).abs() <= (allowed.sum(1) + want.sum(1).abs())).all())


def check(logits, targets, vocab=None, top=0):
    g = gen(99)
    rows, vocab = len(logits), vocab or logits.shape[1]
    gl, gh = torch.randn(rows, generator=g, device=DEV), torch.randn(rows, generator=g, device=DEV)
    want, off = grad64(logits, targets, gl, gh, vocab)
    r = token_logprobs(logits, targets, top=top, vocab=vocab)
    got = token_logprobs_grad(logits, targets, r.lse, r.entropy, gl, gh, vocab=vocab, lse_low=r.lse_low)
    assert got.dtype == logits.dtype
    near(got, want, off)
    leaf = logits.clone().requires_grad_()
    a = token_logprobs(leaf, targets, top=top, vocab=vocab)
    ((a.logprob * gl).sum() + (a.entropy * gh).sum()).backward()
    assert leaf.grad.dtype == logits.dtype and torch.equal(leaf.grad, got)
    inside = logits.clone()
    out = token_logprobs_grad(inside, targets, r.lse, r.entropy, gl, gh, vocab=vocab, out=inside, lse_low=r.lse_low)
    assert out.data_ptr() == inside.data_ptr() and torch.equal(inside, got)
    return r


@pytest.mark.parametrize("offset", [0.0, 1e3, 1e4, 1e5, 1e6, -1e3, -1e6, 3e7])
@pytest.mark.parametrize("rows,columns", [(3, 7), (6, 5000), (2, 40000), (300, 1001)])
def test_common_offsets(rows, columns, offset):
    g = gen(1)
    logits = torch.randn(rows, columns, generator=g, device=DEV) * 2.5 + offset
    targets = torch.randint(0, columns, (rows,), generator=g, device=DEV)
    targets[0] = -100
    r = check(logits, targets, top=3)
    # the pair is the log of the sum, to the sums' own error
    m = logits.double().amax(1, keepdim=True)
    lse = (logits.double() - m).exp().sum(1).log() + m[:, 0]
    assert bool(((r.lse.double() + r.lse_low.double() - lse).abs() <= (columns / 256 + 64) * u).all())


@pytest.mark.parametrize("dtype,offset", [(BF16, 300.0), (BF16, -1e5), (F16, 2000.0), (F16, -6e4)])
@pytest.mark.parametrize("rows,columns", [(4, 300), (2, 40000)])
def test_narrow_types(rows, columns, dtype, offset):
    g = gen(2)
    logits = (torch.randn(rows, columns, generator=g, device=DEV) * 2.5 + offset).to(dtype)
    check(logits, torch.randint(0, columns, (rows,), generator=g, device=DEV))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("columns", [5, 3000, 40000])
def test_rows_of_the_lowest_value(dtype, columns):
    """All logits masked with the type's lowest value are equal: p_j = 1/V."""
    logits = torch.full((3, columns), torch.finfo(dtype).min, dtype=dtype, device=DEV)
    logits[1, 2] = 1.0
    check(logits, torch.tensor([0, 2, -1], device=DEV))


@pytest.mark.parametrize("size", [1e8, 1e30, 3e38])
def test_equal_large_logits(size):
    logits = torch.full((4, 5000), size, device=DEV)
    logits[1, ::3] = -size
    logits[2, 7:] = -math.inf
    check(logits, torch.tensor([0, 1, 3, 4], device=DEV))


def test_padded_columns():
    g = gen(3)
    logits = torch.randn(40, 1100, generator=g, device=DEV) + 1e5
    logits[:, 900:] = math.nan
    check(logits, torch.randint(0, 900, (40,), generator=g, device=DEV), vocab=900)


def test_rows_without_a_finite_log_sum():
    logits = torch.zeros(4, 100, device=DEV)
    logits[0, 5], logits[1, 6], logits[2] = math.nan, math.inf, -math.inf
    targets = torch.tensor([1, 1, 1, 1], device=DEV)
    r = token_logprobs(logits, targets)
    assert not bool(r.lse_low[:3].any())
    one = torch.ones(4, device=DEV)
    got = token_logprobs_grad(logits, targets, r.lse, r.entropy, one, one, lse_low=r.lse_low)
    assert bool(got[:2].isnan().all()) and not bool(got[2].any()) and bool(got[3].isfinite().all())
    none = token_logprobs(logits[:0], targets[:0])
    assert none.lse_low.shape == (0,)
    assert token_logprobs_grad(logits[:0], targets[:0], none.lse, none.entropy, one[:0], lse_low=none.lse_low).shape == (0, 100)


def test_results_are_still_five():
    logits, targets = torch.randn(3, 10, generator=gen(4), device=DEV), torch.tensor([1, 2, 3], device=DEV)
    r = token_logprobs(logits, targets, top=2)
    logprob, entropy, lse, top_logprob, top_index = r
    assert isinstance(r, TokenLogprobs) and len(r) == 5 and r.lse_low.shape == (3,)
    assert TokenLogprobs(logprob, entropy, lse, top_logprob, top_index).lse_low is None
    # without the pair: what lse alone gives
    one = torch.ones(3, device=DEV)
    alone = token_logprobs_grad(logits, targets, r.lse, r.entropy, one)
    zero = token_logprobs_grad(logits, targets, r.lse, r.entropy, one, lse_low=torch.zeros(3, device=DEV))
    assert torch.equal(alone, zero)
