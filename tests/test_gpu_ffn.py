"""The gated feed-forward block on the GPU against the formulas in 64 bits.

The bounds follow the roundings on the way.  u = 2^-24 is half a unit in the
last place of a float32, U that of the tensors' type.  A sum of n products in 32
bits is off by at most (n + 2) u times the sum of the products' sizes.  The
activations are computed in 32 bits: their exponentials' arguments are rounded,
which leaves a relative (16 + 4 w) u with w the size of the argument.  h, da and
db are rounded to the tensors' type (float16: or by half of 2^-24 below its
normal range), and so is every result.
"""
import math

import pytest
import torch

from suika_amd import GatedFFN, PlanError, gated_ffn, gated_ffn_grad

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {t: torch.finfo(t).eps / 2 for t in (F32, BF16, F16)}
u = U[F32]
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -25}
DEV = "cuda"
NAMES = ("out", "x", "gate", "up", "down")


def rows(gen, r, c, dtype, std, pad=0):
    """r rows of c values, `pad` more between them, the first ones from an odd place on."""
    t = torch.empty(r, c + pad, device=DEV, dtype=dtype)[:, pad // 2:pad // 2 + c]
    return t.copy_(torch.randn(r, c, generator=gen, device=DEV) * std)


def block(tokens, hidden, ffn, dtype, pad=0, seed=0):
    gen = torch.Generator(DEV).manual_seed(seed)
    std = max(hidden, 1) ** -0.5
    return (rows(gen, tokens, hidden, dtype, 1.0, pad), rows(gen, ffn, hidden, dtype, std, pad),
            rows(gen, ffn, hidden, dtype, std, pad), rows(gen, hidden, ffn, dtype, max(ffn, 1) ** -0.5, pad),
            rows(gen, tokens, hidden, dtype, 1e-2, pad))


def act64(a, kind):
    """Value, slope, and the size of the exponentials' arguments."""
    if kind == "gelu":
        p = torch.special.ndtr(a)
        return a * p, p + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi), a * a
    if kind == "silu":
        p = torch.sigmoid(a)
        return a * p, p + a * p * (1 - p), a.abs()
    c = math.sqrt(2 / math.pi)
    z, dz = 2 * c * (a + 0.044715 * a ** 3), 2 * c * (1 + 3 * 0.044715 * a * a)
    p = torch.sigmoid(z)
    return a * p, p + a * p * (1 - p) * dz, 3 * z.abs()


def oracle(x, gate, up, down, dy, kind):
    """Results in 64 bits and how far they may be off, by name."""
    dt = x.dtype
    x, gate, up, down, dy = (t.double() for t in (x, gate, up, down, dy))
    (T, H), F = x.shape, gate.shape[0]

    def rounded(value, off):
        return off + (value.abs() + off) * U[dt] + TINY[dt]

    def product(p, q, off_p, off_q, n, k_first=False):
        """p q^T (or p^T q) and its bound."""
        m = (lambda a, b: a.t() @ b) if k_first else (lambda a, b: a @ b.t())
        off = (n + 2) * u * m(p.abs(), q.abs())
        if off_p is not None:
            off = off + m(off_p, q.abs())
        if off_q is not None:
            off = off + m(p.abs(), off_q)
        return m(p, q), off

    a, off_a = product(x, gate, None, None, H)
    b, off_b = product(x, up, None, None, H)
    f, slope, w = act64(a, kind)
    near = (16 + 4 * w) * u
    off_f = 1.2 * off_a + near * f.abs()
    off_slope = off_a + near * 1.3          # second derivatives are below 1
    h = f * b
    off_h = rounded(h, f.abs() * off_b + b.abs() * off_f + off_f * off_b + 4 * u * h.abs())
    y, off_y = product(h, down, off_h, None, F)
    dh, off_dh = product(dy, down.t(), None, None, H)
    da, db = dh * b * slope, dh * f
    off_da = rounded(da, off_dh * (b * slope).abs() + (dh * slope).abs() * off_b + (dh * b).abs() * off_slope
                     + 6 * u * da.abs())
    off_db = rounded(db, off_dh * f.abs() + dh.abs() * off_f + 4 * u * db.abs())
    dx, off_dx = product(torch.cat([da, db], 1), torch.cat([gate, up]).t(), torch.cat([off_da, off_db], 1), None, 2 * F)
    dg, off_dg = product(da, x, off_da, None, T, True)
    du, off_du = product(db, x, off_db, None, T, True)
    dd, off_dd = product(dy, h, None, off_h, T, True)
    value = dict(zip(NAMES, (y, dx, dg, du, dd)))
    return value, {n: rounded(value[n], o) for n, o in zip(NAMES, (off_y, off_dx, off_dg, off_du, off_dd))}


def assert_near(got, want, off, what):
    assert got.shape == want.shape, what
    bad = (got.double() - want).abs() > off
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()}, " \
        f"worst {float(((got.double() - want).abs() / off).max()):.2f} of the bound"


def check(tokens, hidden, ffn, dtype, kind="silu", pad=0):
    args = block(tokens, hidden, ffn, dtype, pad)
    want, off = oracle(*args, kind)
    *tensors, dy = args
    assert_near(gated_ffn(*tensors, activation=kind), want["out"], off["out"], "out")
    r = gated_ffn(*tensors, activation=kind, keep=True)
    assert isinstance(r, GatedFFN) and r.gate.dtype == F32 and r.gate.shape == r.up.shape == (tokens, ffn)
    assert_near(r.out, want["out"], off["out"], "out, kept")
    for n, g in zip(NAMES[1:], gated_ffn_grad(*tensors, r.gate, r.up, dy, activation=kind)):
        assert g.dtype == dtype
        assert_near(g, want[n], off[n], n)


SIZES = [(1, 8, 8), (1, 1, 1), (2, 33, 7), (15, 64, 40), (16, 512, 64), (17, 130, 66), (33, 520, 30), (64, 1032, 56),
         (65, 96, 200), (100, 7, 129), (128, 128, 64), (129, 136, 264), (255, 72, 513), (260, 640, 384), (1000, 256, 1000)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(size, dtype):
    check(*size, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh"])
@pytest.mark.parametrize("size", [(3, 40, 24), (150, 72, 88)], ids=str)
def test_activations(size, kind, dtype):
    check(*size, dtype, kind)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("pad", [1, 2, 5, 8])
@pytest.mark.parametrize("size", [(5, 64, 48), (140, 264, 136), (70, 33, 21)], ids=str)
def test_strides(size, pad, dtype):
    check(*size, dtype, pad=pad)


@pytest.mark.parametrize("size", [(4096, 2048, 1376), (3000, 776, 4504), (300, 264, 40000)], ids=str)
def test_large_tiles(size):
    check(*size, BF16)


@pytest.mark.parametrize("size", [(0, 16, 8), (5, 0, 8), (5, 16, 0), (0, 0, 0), (200, 16, 0), (200, 0, 16)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_empty(size, dtype):
    check(*size, dtype)


def test_rows_with_nan_or_infinity_stay_alone():
    for tokens in (7, 200):
        x, g, up, d, dy = block(tokens, 64, 48, BF16)
        clean = gated_ffn(x, g, up, d)
        x[3, 5] = math.nan
        x[5, 6] = math.inf
        got = gated_ffn(x, g, up, d)
        others = [i for i in range(tokens) if i not in (3, 5)]
        assert torch.equal(got[others], clean[others])
        assert bool(got[3].isnan().all()) and not bool(got[5].isfinite().any())


def test_far_activations():
    """Gates far below zero are 0, far above the gate itself; nothing overflows on the way."""
    gate = torch.tensor([[-3e4], [-200.0], [-90.0], [90.0], [3e4]], device=DEV)
    up, down, x = torch.ones_like(gate), torch.eye(1, 5, device=DEV).repeat(1, 1), torch.ones(1, 1, device=DEV)
    for kind in ("silu", "gelu", "gelu_tanh"):
        for i in range(5):
            down = torch.zeros(1, 5, device=DEV)
            down[0, i] = 1
            r = gated_ffn(x, gate, up, down, activation=kind, keep=True)
            want = 0.0 if i < 3 else float(gate[i])
            assert abs(float(r.out) - want) <= 1e-30 + 4 * u * want
            grads = gated_ffn_grad(x, gate, up, down, r.gate, r.up, torch.ones(1, 1, device=DEV), activation=kind)
            assert all(bool(t.isfinite().all()) for t in grads)
            assert abs(float(grads[1][i]) - (i >= 3)) <= 1e-30 + 4 * u


def test_shapes_and_autograd():
    x, g, up, d, dy = block(30, 64, 48, BF16)
    r = gated_ffn(x, g, up, d, keep=True)
    want = gated_ffn_grad(x, g, up, d, r.gate, r.up, dy)
    leaves = [x.view(2, 15, 64).clone().requires_grad_()] + [t.clone().requires_grad_() for t in (g, up, d)]
    out = gated_ffn(*leaves)
    assert out.shape == (2, 15, 64) and torch.equal(out.view(30, 64), r.out)
    got = torch.autograd.grad(out, leaves, dy.view(2, 15, 64))
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))
    # a gradient that repeats one value, and only the gradients that are wanted
    leaves[0].requires_grad_(False)
    leaves[3].requires_grad_(False)
    gated_ffn(*leaves).sum().backward()
    assert leaves[0].grad is None and leaves[3].grad is None
    ones = gated_ffn_grad(x, g, up, d, r.gate, r.up, torch.ones_like(dy), wanted=(False, True, True, False))
    assert ones[0] is None and ones[3] is None
    assert torch.equal(leaves[1].grad, ones[1]) and torch.equal(leaves[2].grad, ones[2])
    one = gated_ffn(x[3], g, up, d)
    assert one.shape == (64,) and torch.equal(one, gated_ffn(x[3:4], g, up, d)[0])


def test_gradient_against_differences():
    """Central differences of sum(out * c) in float32, step 2^-6: off by the third
    derivative's step^2 / 6 and by the outputs' roundings over the step."""
    x, g, up, d, c = block(6, 12, 10, F32)
    c = c * 100
    r = gated_ffn(x, g, up, d, keep=True)
    grads = gated_ffn_grad(x, g, up, d, r.gate, r.up, c)
    step = 2.0 ** -6
    gen = torch.Generator(DEV).manual_seed(5)
    for i in range(4):
        way = torch.randn(x.shape if i == 0 else (g, up, d)[i - 1].shape, generator=gen, device=DEV)
        way /= way.norm()

        def at(t):
            args = [x, g, up, d]
            args[i] = args[i] + t * way
            return float((gated_ffn(*args).double() * c.double()).sum())

        slope = (at(step) - at(-step)) / (2 * step)
        third = (at(2 * step) - 2 * at(step) + 2 * at(-step) - at(-2 * step)) / (2 * step ** 3)
        noise = 64 * u * float((r.out.abs() * c.abs()).sum()) / step
        assert abs(slope - float((grads[i].double() * way.double()).sum())) <= abs(third) * step ** 2 / 3 + 8 * noise + 1e-4


def test_same_results_every_time_and_on_other_streams():
    x, g, up, d, dy = block(300, 264, 136, BF16)
    r = gated_ffn(x, g, up, d, keep=True)
    grads = gated_ffn_grad(x, g, up, d, r.gate, r.up, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s = gated_ffn(x, g, up, d, keep=True)
        again = gated_ffn_grad(x, g, up, d, s.gate, s.up, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(r.out, s.out) and all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("tokens", [4, 300])
def test_captured(tokens):
    x, g, up, d, dy = block(tokens, 264, 136, BF16)

    def both():
        r = gated_ffn(x, g, up, d, keep=True)
        return (gated_ffn(x, g, up, d), r.out) + gated_ffn_grad(x, g, up, d, r.gate, r.up, dy)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = both()
    for k in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(DEV).manual_seed(k), device=DEV))
        want = both()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_offsets_beyond_32_bits():
    tokens, hidden, ffn = 2 ** 22 + 3, 1024, 8          # x of 8.6 GB
    gen = torch.Generator(DEV).manual_seed(0)
    x = torch.zeros(tokens, hidden, device=DEV, dtype=BF16)
    for at in (0, 2 ** 21, 2 ** 22 - 1, tokens - 5):
        x[at:at + 4] = torch.randn(4, hidden, generator=gen, device=DEV).to(BF16)
    _, g, up, d, _ = block(1, hidden, ffn, BF16)
    r = gated_ffn(x, g, up, d, keep=True)
    dx, dg, _, _ = gated_ffn_grad(x, g, up, d, r.gate, r.up, x)
    for at in (0, 2 ** 21, 2 ** 22 - 1, tokens - 5):
        part = x[at:at + 4]
        small = gated_ffn(part, g, up, d)
        want, off = oracle(part, g, up, d, part, "silu")
        assert_near(r.out[at:at + 4], want["out"], off["out"], "out")
        assert_near(small, want["out"], off["out"], "out")
        assert_near(dx[at:at + 4], want["x"], off["x"], "x")
    some = x[sorted({at + k for at in (0, 2 ** 21, 2 ** 22 - 1, tokens - 5) for k in range(4)})]
    want, off = oracle(some, g, up, d, some, "silu")
    # as many more products of zeros: nothing is rounded in them
    assert_near(dg, want["gate"], off["gate"], "gate")


def test_refusals():
    x, g, up, d, dy = block(4, 16, 8, BF16)
    for args, word in [((x.float(), g, up, d), "dtype"), ((x, g[:, :15], up, d), "ffn x hidden"),
                       ((x, g, up[:7], d), "ffn x hidden"), ((x, g, up, d.t()), "ffn x hidden"),
                       ((x, g, up, d.t().contiguous().t()), "one distance"), ((x.double(),) + (g.double(),) * 2 + (d.double(),), "dtype"),
                       ((x, g.cpu(), up, d), "not on cuda"), ((x, g[0], up, d), "a matrix")]:
        with pytest.raises(PlanError, match=word):
            gated_ffn(*args)
    with pytest.raises(PlanError, match="activation"):
        gated_ffn(x, g, up, d, activation="relu")
    r = gated_ffn(x, g, up, d, keep=True)
    with pytest.raises(PlanError, match="kept_gate"):
        gated_ffn_grad(x, g, up, d, r.gate.bfloat16(), r.up, dy)
    with pytest.raises(PlanError, match="contiguous"):
        gated_ffn_grad(x, g, up, d, r.gate, r.up.t().contiguous().t(), dy)
    with pytest.raises(PlanError, match="grad_output"):
        gated_ffn_grad(x, g, up, d, r.gate, r.up, dy[:3])
    with pytest.raises(PlanError, match="wanted"):
        gated_ffn_grad(x, g, up, d, r.gate, r.up, dy, wanted=(True,))
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(PlanError, match="forward-mode"):
            gated_ffn(fwd.make_dual(x, x), g, up, d)


# Few tokens of enough rows that a workgroup has up to 12 or 24 of both projections' and
# up to 32 of the last product's.
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [(1, 4100, 40), (3, 40, 3005), (24, 72, 5001), (24, 6001, 40), (50, 72, 5000),
                                  (50, 6000, 33), (40, 136, 3500), (31, 264, 9000)], ids=str)
def test_few_tokens_of_many_rows(size, dtype):
    check(*size, dtype)


@pytest.mark.parametrize("tokens", [4, 150])
@pytest.mark.parametrize("ffn", [13, 16])
def test_an_infinity_does_not_meet_the_padding(ffn, tokens):
    """With positive values a row's infinity gives infinities, whatever ffn is a multiple of."""
    gen = torch.Generator(DEV).manual_seed(7)
    x, g, up, d, dy = (torch.rand(s, generator=gen, device=DEV).add_(0.5).to(BF16)
                       for s in ((tokens, 24), (ffn, 24), (ffn, 24), (24, ffn), (tokens, 24)))
    clean = gated_ffn(x, g, up, d, keep=True)
    before = gated_ffn_grad(x, g, up, d, clean.gate, clean.up, dy)[0]
    dy[1, 3] = math.inf
    dx = gated_ffn_grad(x, g, up, d, clean.gate, clean.up, dy)[0]
    others = [i for i in range(tokens) if i != 1]
    assert bool((dx[1] == math.inf).all()) and torch.equal(dx[others], before[others])
    x[1, 5] = math.inf
    kept = gated_ffn(x, g, up, d, keep=True).out
    assert bool((kept[1] == math.inf).all()) and torch.equal(kept[others], clean.out[others])
    assert bool((gated_ffn(x, g, up, d)[1] == math.inf).all())


def test_slope_of_far_gelu_tanh_gates():
    """A gate whose square is beyond float32 has a slope of 0 or 1."""
    for far in (-1e20, 1e20):
        x, gate = torch.ones(1, 1, device=DEV), torch.tensor([[far]], device=DEV)
        up, down = torch.ones(1, 1, device=DEV), torch.ones(1, 1, device=DEV)
        r = gated_ffn(x, gate, up, down, activation="gelu_tanh", keep=True)
        grads = gated_ffn_grad(x, gate, up, down, r.gate, r.up, torch.ones(1, 1, device=DEV), activation="gelu_tanh")
        assert float(grads[1]) == (far > 0)


@pytest.mark.parametrize("size, dtype", [((4096, 2560, 2300), BF16), ((4100, 2555, 2305), F16), ((2000, 40, 72), BF16),
                                         ((3001, 33, 65), F32)], ids=str)
def test_long_sums_of_several_products(size, dtype):
    """The matrices' gradients over many tokens: the tiles behind whole rounds of 256, or all of few, in parts."""
    check(*size, dtype)


def kernels_of(f):
    """The kernels that a call launches."""
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as p:
        f()
        torch.cuda.synchronize()
    return {e.key for e in p.key_averages()}


# Long sums of few tiles: those of the projections and of dh are split too.
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("size", [(5, 4986, 88), (64, 4100, 33), (70, 4242, 40), (200, 3001, 300), (129, 8192, 64), (300, 2056, 520)],
                         ids=str)
def test_long_sums_of_projections(size, dtype):
    names = kernels_of(lambda: check(*size, dtype))
    for k in ("forward_join_kernel", "backward_join_kernel"):
        assert any(k in n for n in names) or (k == "forward_join_kernel" and size[0] <= 64), k


@pytest.mark.parametrize("tokens", [4, 150])
@pytest.mark.parametrize("ffn", [13, 16])
def test_an_infinity_in_split_sums(ffn, tokens):
    """As in sums that are not split: it stays in its row, and does not meet the padding's zeros."""
    gen = torch.Generator(DEV).manual_seed(8)
    x, g, up, d, dy = (torch.rand(s, generator=gen, device=DEV).add_(0.5).mul_(1 / 64).to(BF16)
                       for s in ((tokens, 4104), (ffn, 4104), (ffn, 4104), (4104, ffn), (tokens, 4104)))
    clean = gated_ffn(x, g, up, d, keep=True)
    before = gated_ffn_grad(x, g, up, d, clean.gate, clean.up, dy)[0]
    dy[1, 3] = math.inf
    dx = gated_ffn_grad(x, g, up, d, clean.gate, clean.up, dy)[0]
    others = [i for i in range(tokens) if i != 1]
    assert bool((dx[1] == math.inf).all()) and torch.equal(dx[others], before[others])
    x[1, 5] = math.inf
    kept = gated_ffn(x, g, up, d, keep=True).out
    assert bool((kept[1] == math.inf).all()) and torch.equal(kept[others], clean.out[others])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens", [1, 16, 17, 32, 33])
def test_few_tokens_that_are_kept(tokens, dtype):
    """Odd rows need no copies for few tokens, and the projections are those that the block's output is of."""
    check(tokens, 1025, 333, dtype, pad=3)
    x, g, up, d, _ = block(tokens, 1025, 333, dtype, 3)
    names = kernels_of(lambda: gated_ffn(x, g, up, d, keep=True))
    assert any("align_kernel" in n for n in names) == (tokens > 32), names
    r = gated_ffn(x, g, up, d, keep=True)
    off = (1025 + 2) * u
    for got, w in ((r.gate, g), (r.up, up)):
        want, size = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
        assert bool(((got.double() - want).abs() <= off * size).all())


@pytest.mark.parametrize("way", [-1, 1])
def test_far_silu_gates_in_32_bits(way):
    """The weight's exponential is off by an ulp (2u) whatever its argument, the sum, the division and the product by u
    each: 5u of the value, and 12u of a slope whose two terms are at most 1.5 times their sum."""
    gate = (torch.linspace(5, 85, 161, device=DEV) * way).view(-1, 1)
    n = gate.shape[0]
    x, up, down = torch.ones(1, 1, device=DEV), torch.ones(n, 1, device=DEV), torch.ones(1, n, device=DEV)
    value, slope, _ = act64(gate.double().view(-1), "silu")
    r = gated_ffn(x, gate, up, down, keep=True)
    assert torch.equal(r.gate.view(-1), gate.view(-1))
    _, dgate, dup, _ = gated_ffn_grad(x, gate, up, down, r.gate, r.up, torch.ones(1, 1, device=DEV))
    assert bool(((dup.view(-1) - value).abs() <= 5 * u * value.abs()).all())
    assert bool(((dgate.view(-1) - slope).abs() <= 12 * u * slope.abs()).all())
    for i in (0, 60, 110, n - 1):
        out = float(gated_ffn(x, gate[i:i + 1], up[:1], down[:, :1]))
        assert abs(out - float(value[i])) <= 5 * u * abs(float(value[i]))



# Two whole rounds of 128 x 128 tiles: of the projections and of dh, of y and dx, and of
# the matrices' gradients.
@pytest.mark.parametrize("size, kernels", [((4000, 40, 2001), ("forward_kernel<float, 128>", "backward_kernel<float, 128>")),
                                           ((4000, 2001, 24), ("product_kernel<float, 128, (sr_tile::Side)0, (sr_tile::Side)0>",
                                                               "product_kernel<float, 128, (sr_tile::Side)0, (sr_tile::Side)1>")),
                                           ((30, 1901, 1400), ("product_kernel<float, 128, (sr_tile::Side)1, (sr_tile::Side)1>",))],
                         ids=str)
def test_large_tiles_of_floats(size, kernels):
    names = kernels_of(lambda: check(*size, F32))
    for k in kernels:
        assert any(k in n for n in names), (k, sorted(n for n in names if "kernel<" in n))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("ffn, thin", [(256, True), (264, False)])
def test_few_kept_tokens_of_wide_blocks(ffn, thin, dtype):
    """Rows that tiles can be loaded from: the way of few tokens up to four times as many rows as columns."""
    check(20, 64, ffn, dtype)
    x, g, up, d, _ = block(20, 64, ffn, dtype)
    assert any("thin_kernel" in n for n in kernels_of(lambda: gated_ffn(x, g, up, d, keep=True))) == thin
