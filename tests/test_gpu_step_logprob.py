"""Token log probabilities and their gradient on the GPU against the formulas
in 64 bits.

u = 2^-24, U(type) half a unit in the last place of the stored type.  A lane
adds up to V/256 exponentials of an error of a few u each, and the lanes are
joined in 8 steps, so the sum is known to S = (V/256 + 64) u of itself; lse to
S + 4u|lse|; a log probability to S + 4u(|x| + |lse|); the entropy, a mean of
at most 2 ln V + 1 in magnitude, to S (2 + 3 ln V).  An lse that is stored in
float32 makes p_j of the gradient exact to S + 6u(|x| + |lse|) of itself.
"""
import math

import pytest
import torch

from suika_amd import PlanError, TokenLogprobs, token_logprobs, token_logprobs_grad

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {t: torch.finfo(t).eps / 2 for t in (F32, BF16, F16)}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -25}
u = U[F32]
DEV = "cuda"
INF = math.inf


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def make(g, rows, columns, dtype, std=2.5, vocab=None):
    logits = (torch.randn(rows, columns, generator=g, device=DEV) * std).to(dtype)
    targets = torch.randint(0, vocab or columns, (rows,), generator=g, device=DEV)
    if rows > 2:
        targets[1] = -100
    return logits, targets


def logp64(x):
    """(ln p, lse): the maximum is taken off first, so that an lse of 1e30 does not swallow the sum's logarithm."""
    m = x.amax(1, keepdim=True)
    rest = (x - m).exp().sum(1, keepdim=True).log()
    return (x - m) - rest, (m + rest)[:, 0]


def reference(logits, targets, top, vocab):
    x = logits[:, :vocab].double()
    logp, lse = logp64(x)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
    t = targets.long()
    chosen = logp.gather(1, t.clamp(0, vocab - 1)[:, None])[:, 0]
    chosen = torch.where(t >= vocab, -INF, chosen)
    chosen = torch.where(t < 0, 0.0, chosen)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return TokenLogprobs(chosen, entropy, lse, logp.gather(1, order), order)


def near(got, want, off):
    want = want.expand_as(got)
    same = (got == want.to(got.dtype)) | (got.isnan() & want.isnan())      # also where want is beyond the type
    ok = same | ((got.double() - want).abs() <= off)
    assert bool(ok.all()), (float((got.double() - want).abs()[~ok].max()), got[~ok][:4], want[~ok][:4])


def check(logits, targets, top, vocab=None):
    got = token_logprobs(logits, targets, top=top, vocab=vocab)
    vocab = vocab or logits.shape[1]
    want = reference(logits, targets, top, vocab)
    S = (vocab / 256 + 64) * u
    size = logits[:, :vocab].double().nan_to_num(0, 0, 0).abs().amax(1)
    lse = want.lse.abs().nan_to_num(0, 0, 0)
    assert all(t.dtype == F32 for t in got[:3])
    near(got.lse, want.lse, S + 4 * u * lse)
    near(got.logprob, want.logprob, S + 4 * u * (size + lse))
    near(got.entropy, want.entropy, S * (2 + 3 * math.log(vocab)))
    if top:
        assert got.top_index.dtype == torch.int64 and torch.equal(got.top_index, want.top_index)
        near(got.top_logprob, want.top_logprob, (S + 4 * u * (size + lse))[:, None])
    else:
        assert got.top_logprob is None and got.top_index is None
    return got


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 2), (5, 7), (2, 8), (130, 255), (7, 300), (3, 2048), (4, 2049),
                                          (2, 8191), (3, 32003), (1, 152064), (5, 152063), (700, 1001)])
def test_logprobs(rows, columns, dtype):
    logits, targets = make(gen(1), rows, columns, dtype)
    for top in (0, 1, 5, 20, 64):
        if top <= columns:
            check(logits, targets if top != 5 else targets.int(), top)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_padded_columns_and_strides(dtype):
    g = gen(2)
    wide = (torch.randn(40, 1100, generator=g, device=DEV) * 3).to(dtype)
    wide[:, 900:] = math.nan                    # never read as tokens
    targets = torch.randint(0, 890, (40,), generator=g, device=DEV)
    check(wide, targets, 7, vocab=900)
    check(wide[:, 5:1000], targets, 7, vocab=893)
    got = token_logprobs(wide.view(4, 10, 1100), targets.view(4, 10), top=3, vocab=900)
    flat = token_logprobs(wide, targets, top=3, vocab=900)
    assert got.logprob.shape == (4, 10) and got.top_index.shape == (4, 10, 3)
    assert torch.equal(got.top_index.view(40, 3), flat.top_index) and torch.equal(got.lse.view(40), flat.lse)
    none = token_logprobs(wide[:0], targets[:0], top=2)
    assert none.logprob.shape == (0,) and none.top_index.shape == (0, 2)
    one = token_logprobs(wide[3], targets[3], vocab=900)
    assert one.logprob.shape == () and float(one.logprob) == float(flat.logprob[3])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,columns", [(3, 40), (2, 5000), (1, 152064), (300, 3001)])
def test_masked_logits(rows, columns, dtype):
    """-inf and the type's lowest value in most columns, all columns, all but
    the first, the last or a few."""
    g = gen(3)
    low = torch.finfo(dtype).min
    for mask in (-INF, low):
        logits, targets = make(g, rows, columns, dtype)
        keep = torch.rand(rows, columns, generator=g, device=DEV) < 0.1
        keep[:, 3] = True
        targets = torch.where(targets >= 0, torch.full_like(targets, 3), targets)
        some = logits.masked_fill(~keep, mask)
        check(some, targets, 20)
        for only in ([0], [columns - 1], [3, 17, columns - 2]):
            few = torch.full_like(logits, mask)
            few[:, only] = logits[:, only]
            check(few, torch.full_like(targets, only[0]), 20)
    full = torch.full_like(logits, -INF)
    got = token_logprobs(full, targets, top=5)
    assert bool((got.lse == -INF).all()) and not bool(got.entropy.any())
    assert bool((got.top_logprob == -INF).all())
    assert torch.equal(got.top_index, torch.arange(5, device=DEV).expand(rows, 5))
    assert torch.equal(got.logprob, torch.where(targets >= 0, -INF, 0.0))
    # nothing but the lowest value: as good as equal
    got = token_logprobs(torch.full_like(logits, low), targets, top=5)
    S = (columns / 256 + 64) * u
    near(got.entropy, torch.full((rows,), math.log(columns), device=DEV, dtype=torch.float64), S * (2 + 3 * math.log(columns)))
    near(got.top_logprob, torch.full((rows, 5), -math.log(columns), device=DEV, dtype=torch.float64), S + 8 * u * math.log(columns))
    assert torch.equal(got.top_index, torch.arange(5, device=DEV).expand(rows, 5))


@pytest.mark.parametrize("value", [0.0, -3.0, 88.0])
@pytest.mark.parametrize("columns", [64, 1025, 40000])
def test_equal_logits(value, columns):
    logits = torch.full((3, columns), value, device=DEV, dtype=BF16)
    logits[1, 50] += 1
    logits[2, ::2] = -value if value else -0.0        # -0 ties with 0
    targets = torch.tensor([0, 50, 1], device=DEV)
    check(logits, targets, 64)


def test_nan_and_infinity():
    g = gen(4)
    for columns in (50, 3000, 152064):
        logits, targets = make(g, 4, columns, F32)
        logits[0, 7], logits[0, 30], logits[1, 9], logits[2, 40] = math.nan, INF, INF, -INF
        targets[:] = 9
        got = token_logprobs(logits, targets, top=6)
        for t in (got.logprob, got.entropy, got.lse, got.top_logprob):
            assert bool(t[:2].isnan().all()) and not bool(t[2:].isnan().any())
        order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :6]
        assert torch.equal(got.top_index, order) and got.top_index[0, 0] == 7 and got.top_index[0, 1] == 30
        alone = token_logprobs(logits[2:], targets[2:], top=6)
        assert torch.equal(alone.lse, got.lse[2:])


@pytest.mark.parametrize("size", [1e4, 1e8, 1e30, 3e38])
def test_large_logits(size):
    """Rows whose spread leaves one token, and rows of near equal large ones."""
    g = gen(5)
    logits = torch.randn(6, 5000, generator=g, device=DEV).clamp(-3, 3) * (size / 3)
    check(logits, torch.arange(6, device=DEV), 10)
    logits = torch.full((4, 5000), size, device=DEV)
    logits[:, ::3] = -size
    check(logits, torch.arange(4, device=DEV), 10)


def test_targets_outside():
    logits, targets = make(gen(6), 6, 100, F32)
    targets = torch.tensor([-1, -2 ** 40, 90, 99, 100, 2 ** 40], device=DEV)
    check(logits, targets, 0, vocab=95)


# ----------------------------------------------------------------- gradient

def grad64(logits, targets, gl, gh, vocab):
    x = logits[:, :vocab].double()
    logp, lse = logp64(x)
    lse = lse[:, None]
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(1, keepdim=True)
    t = targets.long()
    gl = torch.where(t >= 0, gl.double(), 0.0)[:, None]
    gh = gh.double()[:, None]
    spread = torch.where(p > 0, p * (logp + entropy), 0.0)
    grad = -gl * p - gh * spread
    hit = (torch.arange(vocab, device=DEV)[None] == t[:, None])
    grad = grad + gl * hit
    S = (vocab / 256 + 64) * u
    size = x.nan_to_num(0, 0, 0).abs().amax(1, keepdim=True) + lse.abs()
    weight = gl.abs() + gh.abs() * (torch.where(p > 0, logp.abs(), 0.0) + entropy + 1)
    off = p * weight * (S + 6 * u * size) + p * gh.abs() * S * (2 + 3 * math.log(max(vocab, 2))) + 4 * u * gl.abs() * hit
    pad = torch.nn.functional.pad
    return pad(grad, (0, logits.shape[1] - vocab)), pad(off, (0, logits.shape[1] - vocab))


def check_grad(logits, targets, gl, gh, vocab=None, **kw):
    r = token_logprobs(logits, targets, vocab=vocab)
    want, off = grad64(logits, targets, gl, gh, vocab or logits.shape[1])
    got = token_logprobs_grad(logits, targets, r.lse, r.entropy, gl, gh, vocab=vocab, **kw)
    assert got.dtype == want.dtype or got.dtype == kw.get("dtype", got.dtype)
    near(got, want, off + U[got.dtype] * (want.abs() + off) + TINY[got.dtype])
    return got


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 2), (5, 7), (130, 255), (7, 300), (4, 2049), (3, 32003),
                                          (2, 152064), (700, 1001)])
def test_gradient(rows, columns, dtype):
    g = gen(7)
    logits, targets = make(g, rows, columns, dtype)
    gl, gh = torch.randn(rows, generator=g, device=DEV), torch.randn(rows, generator=g, device=DEV)
    before = logits.clone()
    got = check_grad(logits, targets, gl, gh)
    assert torch.equal(logits, before)
    r = token_logprobs(logits, targets)
    zero = torch.zeros(rows, device=DEV)
    for a, b in ((gl, None), (None, gh), (None, None)):
        part = token_logprobs_grad(logits, targets.int(), r.lse, r.entropy, a, b)
        full = token_logprobs_grad(logits, targets, r.lse, r.entropy, zero if a is None else a, zero if b is None else b)
        assert torch.equal(part, full)
    assert token_logprobs_grad(logits, targets, r.lse, r.entropy, gl, gh, out=logits).data_ptr() == logits.data_ptr()
    assert torch.equal(logits, got)


def test_gradient_padded_strided_masked():
    g = gen(8)
    wide = torch.randn(40, 1100, generator=g, device=DEV) * 3
    wide[:, 900:] = math.nan
    wide[torch.rand(40, 1100, generator=g, device=DEV) < 0.5] = -INF
    targets = torch.randint(0, 890, (40,), generator=g, device=DEV)
    wide[torch.arange(40), targets] = 0.5
    wide[6, :900] = -INF                        # an empty row
    gl, gh = torch.randn(40, generator=g, device=DEV), torch.randn(40, generator=g, device=DEV)
    rows = torch.arange(40, device=DEV) != 6
    check_grad(wide[rows], targets[rows], gl[rows], gh[rows], vocab=900)
    room = torch.full((40, 1200), 5.0, device=DEV)
    r = token_logprobs(wide, targets, vocab=900)
    got = token_logprobs_grad(wide, targets, r.lse, r.entropy, gl, gh, vocab=900, out=room[:, 50:1150])
    assert torch.equal(got, room[:, 50:1150]) and not bool(got[:, 900:].any()) and not bool(got[6].any())
    assert bool((room[:, :50] == 5).all()) and bool((room[:, 1150:] == 5).all()) and bool(got.isfinite().all())


def test_gradient_of_nan_rows():
    logits = torch.zeros(2, 64, device=DEV)
    logits[0, 5] = math.nan
    targets = torch.tensor([1, 1], device=DEV)
    r = token_logprobs(logits, targets)
    one = torch.ones(2, device=DEV)
    got = token_logprobs_grad(logits, targets, r.lse, r.entropy, one, one)
    assert bool(got[0].isnan().all()) and bool(got[1].isfinite().all())


def test_autograd():
    g = gen(9)
    logits, targets = make(g, 12, 500, F32)
    gl, gh = torch.randn(12, generator=g, device=DEV), torch.randn(12, generator=g, device=DEV)
    want, off = grad64(logits, targets, gl, gh, 490)
    logits.requires_grad_()
    r = token_logprobs(logits.view(3, 4, 500), targets.view(3, 4), top=3, vocab=490)
    assert not r.lse.requires_grad and not r.top_logprob.requires_grad
    ((r.logprob.view(-1) * gl).sum() + (r.entropy.view(-1) * gh).sum()).backward()
    near(logits.grad, want, off + 2 * u * want.abs())
    logits.grad = None
    token_logprobs(logits, targets).logprob.sum().backward()
    want, off = grad64(logits.detach(), targets, torch.ones(12, device=DEV), torch.zeros(12, device=DEV), 500)
    near(logits.grad, want, off + 2 * u * want.abs())
    logits.grad = None
    token_logprobs(logits, targets).entropy.sum().backward()
    assert logits.grad is not None
    with torch.no_grad():
        assert not token_logprobs(logits, targets).logprob.requires_grad


def test_gradient_against_differences():
    """Along a direction D, f(x + hD) - f(x - hD) = 2h <grad, D> + O(h^3); the
    values come with the roundings of the log probabilities (S + 4u(|x| +
    |lse|), entropies S (2 + 3 ln V)), the third derivatives are below
    8 |D|^3 (1 + ln V) for logits that are moved by |D| at most."""
    g = gen(10)
    rows, vocab = 20, 1000
    logits, targets = make(g, rows, vocab, F32, std=1.0)
    D = torch.rand(rows, vocab, generator=g, device=DEV) * 2 - 1
    h = 2.0 ** -5
    one = torch.ones(rows, device=DEV)
    r = token_logprobs(logits, targets)
    plus, minus = token_logprobs(logits + h * D, targets), token_logprobs(logits - h * D, targets)
    S = (vocab / 256 + 64) * u
    size = float(logits.abs().max()) + 1 + float(r.lse.abs().max())
    third = 8 * h ** 3 * (1 + math.log(vocab))
    for f, grads, bound in (("logprob", (one, None), S + 8 * u * size), ("entropy", (None, one), S * (2 + 3 * math.log(vocab)))):
        slope = (token_logprobs_grad(logits, targets, r.lse, r.entropy, *grads).double() * D.double()).sum(1)
        change = getattr(plus, f).double() - getattr(minus, f).double()
        assert bool(((change - 2 * h * slope).abs() <= 2 * bound + third).all())
        assert float((change.abs() > 4 * bound).float().mean()) > 0.5      # the change is well above the roundings


def test_refusals():
    logits = torch.zeros(4, 10, device=DEV)
    targets = torch.zeros(4, dtype=torch.int64, device=DEV)
    r = token_logprobs(logits, targets)
    one = torch.ones(4, device=DEV)
    for call, match in [
            (lambda: token_logprobs(logits, targets[:3]), "targets' shape"),
            (lambda: token_logprobs(logits, targets.float()), "int64 or int32"),
            (lambda: token_logprobs(logits, targets.cpu()), "cpu"),
            (lambda: token_logprobs(logits.double(), targets), "Double"),
            (lambda: token_logprobs(logits, targets, top=11), "top 11"),
            (lambda: token_logprobs(logits, targets, top=-1), "top -1"),
            (lambda: token_logprobs(torch.zeros(4, 100, device=DEV), targets, top=65), "at most 64"),
            (lambda: token_logprobs(logits, targets, vocab=0), "vocabulary of 0"),
            (lambda: token_logprobs(logits, targets, vocab=11), "vocabulary of 11"),
            (lambda: token_logprobs(logits.t().contiguous().t(), targets), "dense elements"),
            (lambda: token_logprobs(logits[:1].expand(4, 10), targets), "dense elements"),
            (lambda: token_logprobs(logits, targets.repeat(2)[::2]), "contiguous targets"),
            (lambda: token_logprobs_grad(logits, targets, r.lse.double(), r.entropy, one), "lse"),
            (lambda: token_logprobs_grad(logits, targets, r.lse, r.entropy[:3], one), "entropy"),
            (lambda: token_logprobs_grad(logits, targets, r.lse, r.entropy, one.bfloat16()), "grad_logprob"),
            (lambda: token_logprobs_grad(logits, targets, r.lse, r.entropy, one, one.cpu()), "grad_entropy"),
            (lambda: token_logprobs_grad(logits, targets, r.lse, r.entropy, one, out=logits.half()), "out"),
            (lambda: token_logprobs_grad(logits[:, 1:], targets, r.lse, r.entropy, one, out=logits[:, :9]), "overlaps")]:
        with pytest.raises(PlanError, match=match):
            call()


def test_on_another_stream_and_in_a_graph():
    g = gen(11)
    logits, targets = make(g, 8, 20000, BF16)
    gl, gh = torch.randn(8, generator=g, device=DEV), torch.randn(8, generator=g, device=DEV)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        r = token_logprobs(logits, targets, top=9)
        grad = token_logprobs_grad(logits, targets, r.lse, r.entropy, gl, gh)
    for k in range(3):
        logits.copy_(make(g, 8, 20000, BF16)[0])
        if k == 1:
            logits[2] = 1.0
        graph.replay()
        torch.cuda.synchronize()
        e = token_logprobs(logits, targets, top=9)
        for a, b in zip(r, e):
            assert torch.equal(a, b)
        assert torch.equal(grad, token_logprobs_grad(logits, targets, e.lse, e.entropy, gl, gh))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = token_logprobs(logits, targets, top=9)
    side.synchronize()
    assert torch.equal(again.lse, e.lse) and torch.equal(again.top_index, e.top_index)
