"""Embedding of a vocabulary shard and its gradient on the GPU against plain
forms in 64 bits.

u = 2^-24 is half a unit in the last place of a float32, U(type) of the stored
type.  A looked-up element is rounded as scale, as product and where it is
stored: 2u + U.  A row's gradient of n tokens is a sum of n terms in 32 bits,
in some order: (n + 2) u times the sum of the magnitudes, and U of the result.
"""
import pytest
import torch

from suika_amd import PlanError, vocab_embedding, vocab_embedding_grad

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {t: torch.finfo(t).eps / 2 for t in (F32, BF16, F16)}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -25}
u = U[F32]
DEV = "cuda"


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def some_tokens(g, n, low, high, dtype=torch.int64):
    return torch.randint(low, high, (n,), generator=g, device=DEV, dtype=torch.int64).to(dtype)


def lookup64(tokens, weight, scale, start):
    at = tokens.long().reshape(-1) - start
    inside = (at >= 0) & (at < len(weight))
    rows = weight.double()[at.clamp(0, len(weight) - 1)] * scale
    return torch.where(inside[:, None], rows, 0.0)


def grad64(tokens, grad_out, rows, scale, start):
    """(gradient, how far a float32 sum of the terms may be off)"""
    at = tokens.long().reshape(-1) - start
    spare = torch.where((at >= 0) & (at < rows), at, rows)
    g = grad_out.double().reshape(len(spare), grad_out.shape[-1])
    total = torch.zeros(rows + 1, g.shape[1], dtype=torch.float64, device=DEV)
    total.index_add_(0, spare, g)
    size = torch.zeros_like(total).index_add_(0, spare, g.abs())
    n = torch.bincount(spare, minlength=rows + 1)[:rows, None]
    return total[:rows] * scale, (n + 2) * u * size[:rows] * abs(scale)


def assert_near(got, want, off):
    dt = got.dtype
    allowed = off + U[dt] * (want.abs() + off) + TINY[dt]
    diff = (got.double() - want).abs()
    assert got.shape == want.shape
    assert bool((diff <= allowed).all()), (float(diff.max()), float((diff / allowed).max()))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [1, 3, 8, 60, 257, 2049, 4096, 8200])
@pytest.mark.parametrize("n,token_dtype", [(1, torch.int64), (67, torch.int32), (1000, torch.int64)])
def test_lookup(n, token_dtype, cols, dtype):
    g = gen(1)
    weight = randn(g, 50, cols, dtype=dtype)
    tokens = some_tokens(g, n, 80, 170, token_dtype)     # the shard is 100..150: some on either side
    got = vocab_embedding(tokens, weight, scale=1.7, vocab_start=100)
    want = lookup64(tokens, weight, 1.7, 100)
    assert got.dtype == dtype and got.shape == (n, cols)
    assert_near(got, want, 2 * u * want.abs())
    plain = vocab_embedding(tokens - 100, weight)
    assert torch.equal(plain, lookup64(tokens, weight, 1.0, 100).to(dtype))     # a scale of 1 copies


def test_lookup_shapes_strides_and_out():
    g = gen(2)
    table = randn(g, 40, 100, dtype=BF16)
    weight = table[:, 3:90]                              # rows 100 apart, at odd addresses
    tokens = some_tokens(g, 24, 0, 40).view(2, 3, 4)
    got = vocab_embedding(tokens, weight)
    assert got.shape == (2, 3, 4, 87) and torch.equal(got, weight[tokens])
    out = torch.zeros(2, 3, 4, 87, device=DEV, dtype=BF16)
    v = out._version
    assert vocab_embedding(tokens, weight, out=out) is out or torch.equal(out, got)
    assert torch.equal(out, got) and out._version > v
    assert vocab_embedding(tokens[:0], weight).shape == (0, 3, 4, 87)
    assert torch.equal(vocab_embedding(tokens[0, 0, 0], weight), weight[tokens[0, 0, 0]])
    empty = vocab_embedding(tokens, weight[:0])
    assert empty.shape == (2, 3, 4, 87) and not bool(empty.any())
    far = torch.tensor([2 ** 62, -2 ** 62, -1, 39], device=DEV)
    assert torch.equal(vocab_embedding(far, weight), torch.cat([torch.zeros(3, 87, device=DEV, dtype=BF16), weight[39:40]]))


SIZES = [(0, 5, 8), (1, 1, 1), (63, 3, 60), (64, 1, 16), (65, 1, 33), (129, 300, 7), (1000, 257, 64), (2049, 4, 130),
         (5000, 16000, 24), (20011, 7, 96), (40000, 3000, 8)]


@pytest.mark.parametrize("n,rows,cols", SIZES)
@pytest.mark.parametrize("dtype,grad_dtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F32, BF16)])
def test_grad(n, rows, cols, dtype, grad_dtype):
    g = gen(3)
    start = 10
    tokens = some_tokens(g, n, start - 2, start + rows + 2)
    heavy = torch.rand(n, generator=g, device=DEV) < 0.3         # one token of many, as a filler is
    tokens = torch.where(heavy, torch.full_like(tokens, start + rows // 2), tokens)
    grad_out = randn(g, n, cols, dtype=dtype)
    got = vocab_embedding_grad(tokens, grad_out, rows, scale=0.5, vocab_start=start, dtype=grad_dtype)
    want, off = grad64(tokens, grad_out, rows, 0.5, start)
    assert got.dtype == grad_dtype
    assert_near(got, want, off)
    again = vocab_embedding_grad(tokens.int(), grad_out, rows, scale=0.5, vocab_start=start, dtype=grad_dtype)
    assert torch.equal(got, again)


@pytest.mark.parametrize("n", [33, 64, 65, 66, 96, 97, 4097, 16384, 16385, 70000])
def test_grad_of_one_token(n):
    """All tokens in one row: cut into pieces and joined."""
    g = gen(4)
    grad_out = randn(g, n, 12, dtype=BF16)
    tokens = torch.full((n,), 3, device=DEV)
    want, off = grad64(tokens, grad_out, 5, 1.0, 0)
    assert_near(vocab_embedding_grad(tokens, grad_out, 5, dtype=F32), want, off)


def test_grad_rows_of_every_length():
    """Rows of 0, 1, 2, ... 130 tokens in mixed order: short rows, cut rows and
    what the pieces leave over."""
    g = gen(5)
    tokens = torch.repeat_interleave(torch.arange(131, device=DEV), torch.arange(131, device=DEV))
    tokens = tokens[torch.randperm(len(tokens), generator=g, device=DEV)]
    grad_out = randn(g, len(tokens), 40)
    want, off = grad64(tokens, grad_out, 131, 1.0, 0)
    assert_near(vocab_embedding_grad(tokens, grad_out, 131), want, off)


@pytest.mark.parametrize("grad_dtype", [F32, BF16])
def test_grad_accumulates(grad_dtype):
    g = gen(6)
    tokens = some_tokens(g, 700, 0, 30)
    tokens[:300] = 7
    grad_out = randn(g, 700, 50, dtype=BF16)
    out = randn(g, 60, 50, dtype=grad_dtype)
    out[45] = float("nan")                               # a row without tokens is not touched
    old = out.clone()
    got = vocab_embedding_grad(tokens, grad_out, 60, scale=2.0, out=out, accumulate=True)
    want, off = grad64(tokens, grad_out, 60, 2.0, 0)
    assert got.data_ptr() == out.data_ptr()
    rows = torch.arange(60, device=DEV) != 45
    assert_near(out[rows], (want + old.double())[rows], (off + u * (want.abs() + old.double().abs()))[rows])
    assert bool(out[45].isnan().all())
    vocab_embedding_grad(tokens, grad_out, 60, out=out)
    want, off = grad64(tokens, grad_out, 60, 1.0, 0)
    assert_near(out, want, off)


@pytest.mark.parametrize("cols", [5, 511, 999, 2047, 2053, 4100])
@pytest.mark.parametrize("dtype,grad_dtype", [(BF16, F32), (F16, F16), (F32, F32)])
def test_grad_of_wide_rows_and_their_ends(cols, dtype, grad_dtype):
    """Rows that take part of a wave, whole waves or a workgroup twice over, with
    a last block that is not whole; short, long and cut, added to what is there."""
    g = gen(8)
    lengths = torch.tensor([0, 1, 2, 3, 9, 10, 17, 32, 33, 300, 900], device=DEV)
    tokens = torch.repeat_interleave(torch.arange(len(lengths), device=DEV), lengths)
    tokens = tokens[torch.randperm(len(tokens), generator=g, device=DEV)]
    grad_out = randn(g, len(tokens), cols, dtype=dtype)
    out = randn(g, len(lengths), cols, dtype=grad_dtype)
    old = out.double()
    want, off = grad64(tokens, grad_out, len(lengths), 0.5, 0)
    vocab_embedding_grad(tokens, grad_out, len(lengths), scale=0.5, out=out, accumulate=True)
    assert_near(out, want + old, off + u * (want.abs() + old.abs()))
    vocab_embedding_grad(tokens, grad_out, len(lengths), scale=0.5, out=out)
    assert_near(out, want, off)


def test_grad_strides_and_shapes():
    g = gen(7)
    wide = randn(g, 90, 70, dtype=BF16)
    tokens = some_tokens(g, 90, 0, 9)
    want, off = grad64(tokens, wide[:, 5:38], 9, 1.0, 0)
    assert_near(vocab_embedding_grad(tokens, wide[:, 5:38], 9), want, off)
    shaped = randn(g, 3, 30, 33)
    want, off = grad64(tokens, shaped, 9, 1.0, 0)
    assert_near(vocab_embedding_grad(tokens.view(3, 30), shaped, 9), want, off)
    assert vocab_embedding_grad(tokens, wide, 0).shape == (0, 70)


def test_non_finite_gradients_stay_in_their_rows():
    tokens = torch.tensor([0, 1, 2, 99, 1], device=DEV)
    grad_out = torch.ones(5, 20, device=DEV)
    grad_out[0, 3], grad_out[3, 4] = float("inf"), float("nan")
    got = vocab_embedding_grad(tokens, grad_out, 4)
    assert bool(got[0, 3].isinf()) and int((~got.isfinite()).sum()) == 1
    assert float(got[1, 0]) == 2 and not bool(got[3].any())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_autograd_and_differences(dtype):
    """The backward pass gives the formula's gradient, and the loss's change
    along a direction is the gradient's product with it (the operator is
    linear in the weight, so the difference is exact but for roundings)."""
    g = gen(8)
    weight = randn(g, 30, 24, dtype=dtype).requires_grad_()
    tokens = some_tokens(g, 100, 0, 40).view(4, 25)
    factor = randn(g, 4, 25, 24, dtype=dtype)
    out = vocab_embedding(tokens, weight, scale=3.0, vocab_start=5)
    out.backward(factor)
    want, off = grad64(tokens, factor, 30, 3.0, 5)
    assert weight.grad.dtype == dtype
    assert_near(weight.grad, want, off)
    if dtype == F32:
        direction = randn(g, 30, 24)
        with torch.no_grad():
            there = vocab_embedding(tokens, weight + direction, scale=3.0, vocab_start=5)
            change = ((there.double() - out.detach().double()) * factor.double()).sum()
        slope = (weight.grad.double() * direction.double()).sum()
        size = (there.double().abs() + out.detach().double().abs()).mul(factor.double().abs()).sum() + \
            (off + u * want.abs()).mul(direction.double().abs()).sum() / u
        assert abs(float(change - slope)) <= 4 * u * float(size)
    with torch.no_grad():
        assert not vocab_embedding(tokens, weight).requires_grad
    # an expanded gradient, as a sum's backward gives
    weight.grad = None
    vocab_embedding(tokens, weight).sum().backward()
    ones, off = grad64(tokens, torch.ones(100, 24, device=DEV), 30, 1.0, 0)
    assert_near(weight.grad, ones, off)


def test_shards_add_up_to_the_embedding():
    g = gen(9)
    whole = randn(g, 64, 16, dtype=BF16)
    tokens = some_tokens(g, 200, 0, 64)
    parts = [vocab_embedding(tokens, whole[16 * i:16 * i + 16], vocab_start=16 * i) for i in range(4)]
    assert torch.equal(sum(p.float() for p in parts).to(BF16), whole[tokens])


def test_refusals():
    tokens = torch.zeros(4, dtype=torch.int64, device=DEV)
    weight = torch.zeros(5, 6, device=DEV)
    grad_out = torch.zeros(4, 6, device=DEV)
    for call, match in [
            (lambda: vocab_embedding(tokens.float(), weight), "int64 or int32"),
            (lambda: vocab_embedding(tokens.repeat(2)[::2], weight), "contiguous"),
            (lambda: vocab_embedding(tokens, weight.double()), "Double"),
            (lambda: vocab_embedding(tokens, weight.cpu()), "cpu"),
            (lambda: vocab_embedding(tokens, weight.t()), "dense elements"),
            (lambda: vocab_embedding(tokens, weight[:1].expand(5, 6)), "dense elements"),
            (lambda: vocab_embedding(tokens, weight, out=torch.zeros(4, 5, device=DEV)), "out"),
            (lambda: vocab_embedding(tokens, weight, out=torch.zeros(4, 6, device=DEV, dtype=BF16)), "out"),
            (lambda: vocab_embedding(tokens, weight, out=weight[:4]), "overlaps"),
            (lambda: vocab_embedding_grad(tokens, grad_out[:3], 5), "tokens' shape"),
            (lambda: vocab_embedding_grad(tokens, grad_out, -1), "rows"),
            (lambda: vocab_embedding_grad(tokens, grad_out, 5, dtype=torch.float64), "Double"),
            (lambda: vocab_embedding_grad(tokens, grad_out, 5, accumulate=True), "goes with out"),
            (lambda: vocab_embedding_grad(tokens, grad_out, 5, out=torch.zeros(4, 6, device=DEV)), "rows x columns"),
            (lambda: vocab_embedding_grad(tokens, grad_out, 5, dtype=BF16, out=weight), "another dtype"),
            (lambda: vocab_embedding_grad(tokens, grad_out, 4, out=grad_out), "overlaps"),
            (lambda: vocab_embedding_grad(tokens, grad_out.t().contiguous().t(), 5), "dense elements")]:
        with pytest.raises(PlanError, match=match):
            call()


def test_on_another_stream_and_in_a_graph():
    g = gen(10)
    tokens = some_tokens(g, 3000, 0, 500)
    tokens[:900] = 11
    grad_out = randn(g, 3000, 64, dtype=BF16)
    weight = randn(g, 400, 64, dtype=BF16)
    want = vocab_embedding_grad(tokens, grad_out, 400)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = vocab_embedding_grad(tokens, grad_out, 400)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        rows = vocab_embedding(tokens, weight)
        got = vocab_embedding_grad(tokens, grad_out, 400)
    for k in range(3):
        tokens.copy_(some_tokens(g, 3000, 0, 500))
        tokens[:800 * k] = 3 + k
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(rows, vocab_embedding(tokens, weight))
        assert torch.equal(got, vocab_embedding_grad(tokens, grad_out, 400))
