"""Newton-Schulz products and the Muon update on the GPU against 64 bits.

A step's operands are held in 22 bits and its three products summed in 32, with
roundings that add up like independent ones: together 4 * 2^-22 of the result's
size at most.  What is rounded in a step grows by the polynomial's largest slope,
its first coefficient (3.4445), in each later one, so after k steps the result's
distance from the exact one, both as norms of all elements, is at most 3.4445^k
2^-20, and its own rounding U of what is stored.  A momentum is two products and
a sum in 32 bits: 3u of their sizes; a weight adds its decay and the update.
"""
import math
import threading

import pytest
import torch

from suika_amd import PlanError, ShardMuon, grad_norm, grad_square_sum, orthogonalize
from suika_amd.muon import COEFFICIENTS

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {t: torch.finfo(t).eps / 2 for t in (F32, BF16, F16)}
u = U[F32]
DEV = "cuda"


def growth(steps):
    return COEFFICIENTS[0] ** steps * 2.0 ** -20


def exact(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    x = g.double()
    x = x / x.norm().clamp(min=eps)
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    rows = [coefficients] * steps if isinstance(coefficients[0], float) else coefficients
    for a, b, c in rows:
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if flip else x


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def draw(shape, kind="normal", dtype=F32, seed=0, std=1.0):
    g = gen(seed)
    r, c = shape
    x = torch.randn(r, c, generator=g, device=DEV)
    if kind == "low rank":
        k = max(1, min(r, c) // 8)
        x = 0.01 * x + torch.randn(r, k, generator=g, device=DEV) @ torch.randn(k, c, generator=g, device=DEV)
    return (x * std).to(dtype)


def near(got, want, steps=5, what=""):
    dt = got.dtype
    off = float((got.double() - want).norm())
    size = float(want.norm())
    assert off <= (growth(steps) + U[dt]) * size, f"{what}: {off / max(size, 1e-300):.2e} off, {growth(steps) + U[dt]:.2e} allowed"


SHAPES = [(1, 1), (1, 2), (1, 300), (300, 1), (2, 3), (7, 5), (16, 16), (24, 16), (31, 33), (33, 31), (32, 64), (64, 64), (64, 65), (64, 200),
          (3133, 4), (5, 3000), (3200, 4), (16, 784), (785, 16), (32, 256), (257, 32), (63, 61),
          (65, 64), (100, 300), (127, 130), (128, 128), (129, 257), (200, 1000), (1000, 200), (256, 320), (300, 299), (520, 530)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_shapes(shape, dtype):
    g = draw(shape, dtype=dtype)
    before = g.clone()
    for steps in (1, 2, 5):
        out, = orthogonalize([g], steps=steps)
        assert out.shape == g.shape and out.dtype == dtype and out.is_contiguous()
        near(out, exact(g, steps), steps, f"{steps} steps")
    assert torch.equal(g, before)


@pytest.mark.parametrize("shape", [(64, 200), (300, 130), (512, 512)], ids=str)
def test_low_rank(shape):
    g = draw(shape, "low rank")
    near(orthogonalize([g])[0], exact(g))


def test_lists():
    """Small, large, wide and tall ones at once, more than a launch's table takes."""
    shapes = (SHAPES + [(0, 5), (5, 0), (700, 1500)]) * 3
    gs = [draw(s, dtype=(F32, BF16, F16)[i % 3], seed=i) for i, s in enumerate(shapes)]
    out = orthogonalize(gs)
    for i, (g, o) in enumerate(zip(gs, out)):
        assert o.shape == g.shape and o.dtype == g.dtype
        if g.numel():
            near(o, exact(g), what=f"{i}: {tuple(g.shape)}")
    assert all(torch.equal(a, b) for a, b in zip(out, orthogonalize(tuple(gs))))
    # alone or in a list: the same products, in tiles that may have other sizes
    near(orthogonalize([gs[30]])[0], out[30].double())
    assert orthogonalize([]) == []


def test_large():
    gs = [draw(s, seed=i, dtype=BF16) for i, s in enumerate([(2048, 4096), (4096, 1030), (2500, 2300)])]
    for g, o in zip(gs, orthogonalize(gs)):
        near(o, exact(g))


def test_strides_and_outputs():
    for shape in ((70, 90), (200, 130)):
        wide = draw((shape[0], shape[1] + 7))
        g = wide[:, 3:3 + shape[1]]
        want = exact(g)
        near(orthogonalize([g])[0], want)
        out = torch.full((shape[0], shape[1] + 5), 9.0, device=DEV, dtype=BF16)
        inner = out[:, 2:-3]
        version = out._version
        got, = orthogonalize([g], out=[inner])
        assert got is not None and got.data_ptr() == inner.data_ptr() and out._version > version
        near(inner, want)
        assert bool((out[:, :2] == 9).all()) and bool((out[:, -3:] == 9).all())
        same = g.clone()
        orthogonalize([same], out=[same])
        near(same, want)


def test_sizes_of_values():
    """The scale of a matrix does not matter, from float32's smallest to its largest."""
    g = draw((70, 90))
    want = orthogonalize([g])[0]
    for scale in (2.0 ** -100, 2.0 ** 100):
        got, = orthogonalize([g * scale], eps=0.0)
        assert torch.equal(got, want)
    # below eps a matrix is divided by eps only
    near(orthogonalize([g * 1e-9], eps=1e-3)[0], exact(g * 1e-9, eps=1e-3))


def test_zeros_nan_and_infinity():
    for size in (20, 200):
        good, zero = draw((size, size + 10)), torch.zeros(size, size + 3, device=DEV)
        bad, far = draw((size, size), seed=1), draw((size + 40, size), seed=2)
        bad[size // 2, 3] = math.nan
        far[0, 0] = math.inf
        a, z, b, f, c = orthogonalize([good, zero, bad, far, good])
        assert torch.equal(a, c) and torch.equal(a, orthogonalize([good, zero, zero, zero, good])[0])
        assert bool((orthogonalize([zero], eps=0.0)[0] == 0).all())
        near(a, exact(good))
        assert bool((z == 0).all()) and bool(b.isnan().all()) and bool(f.isnan().all())


def test_other_coefficients():
    g = draw((96, 160))
    schedule = [(3.9, -7.1, 4.1), (2.9, -3.1, 1.1), (1.875, -1.25, 0.375)]
    got, = orthogonalize([g], steps=3, coefficients=schedule)
    off = float((got.double() - exact(g, 3, schedule)).norm())
    # slopes up to 3.9, 2.9 and 1.875
    assert off <= 3.9 * 2.9 * 1.875 * 2.0 ** -20 * float(got.norm())
    g = draw((40, 50))
    cubic, = orthogonalize([g], steps=12, coefficients=(1.5, -0.5, 0.0))
    off = float((cubic.double() - exact(g, 12, (1.5, -0.5, 0.0))).norm())
    assert off <= 1.5 ** 12 * 2.0 ** -20 * float(cubic.norm())


def test_refusals():
    g = draw((8, 8))
    for kw, word in [(dict(steps=0), "steps"), (dict(coefficients=(2.0, 0.0, 0.0)), "range"), (dict(out=[]), "out has"),
                     (dict(out=[g.t()[:4]]), "one distance|shape"), (dict(out=[draw((8, 9))]), "shape"),
                     (dict(split=[0]), "no reduce"), (dict(split=[2], all_reduce=print), "None, 0 or 1")]:
        with pytest.raises(PlanError, match=word):
            orthogonalize([g], **kw)
    with pytest.raises(PlanError, match="wants a gradient"):
        orthogonalize([g.clone().requires_grad_()])
    with torch.no_grad():
        assert torch.equal(orthogonalize([g.clone().requires_grad_()])[0], orthogonalize([g])[0])
    with pytest.raises(PlanError, match="a matrix"):
        orthogonalize([g[0]])
    with pytest.raises(PlanError, match="dtype"):
        orthogonalize([g.double()])
    with pytest.raises(PlanError, match="not on the GPU"):
        orthogonalize([g, g.cpu()])
    with pytest.raises(PlanError, match="not a tensor"):
        orthogonalize([g, None])
    with pytest.raises(PlanError, match="one distance"):
        orthogonalize([draw((8, 9)).t()])


def test_captured():
    gs = [draw(s) for s in ((20, 30), (150, 200), (300, 260))]
    orthogonalize(gs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = orthogonalize(gs)
    for k in range(4):
        for i, g in enumerate(gs):
            g.copy_(draw(tuple(g.shape), seed=10 * k + i))
        want = orthogonalize(gs)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want))


# ------------------------------------------------------------------ ranks

class Ranks:
    """Ranks as threads of this process, one after another on one GPU."""

    def __init__(self, n):
        self.n, self.given = n, [None] * n
        self.barrier = threading.Barrier(n, timeout=60)
        self.calls = [0] * n

    def all_reduce(self, rank):
        def f(t):
            assert t.dim() == 1 and t.dtype in (F32, torch.float64) and t.device.type == "cuda"
            self.calls[rank] += 1
            self.given[rank] = t
            self.barrier.wait()
            total = sum(x.clone() for x in self.given)
            torch.cuda.synchronize()
            self.barrier.wait()
            t.copy_(total)
            torch.cuda.synchronize()
            self.barrier.wait()
        return f

    def run(self, f):
        out, errors = [None] * self.n, []

        def work(r):
            try:
                out[r] = f(r, self.all_reduce(r))
            except BaseException as e:
                errors.append(e)
                self.barrier.abort()

        threads = [threading.Thread(target=work, args=(r,)) for r in range(self.n)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        if errors:
            raise errors[0]
        return out


@pytest.mark.parametrize("n", [2, 3])
def test_split(n):
    """Parts of matrices by rows and by columns, uneven ones and an empty one, with whole ones beside them."""
    shapes = [(96, 40), (40, 96), (130, 300), (300, 130), (64, 64)]
    splits = [0, 1, 0, 1, None]
    gs = [draw(s, seed=i) for i, s in enumerate(shapes)] + [draw((2, 30), seed=9)]
    splits.append(0)

    def parts(g, d, r):
        if d is None:
            return g
        if g.shape[0] == 2:
            return g[r:r + 1] if r < 2 else g[:0]         # nothing is left for a third rank
        cut = [0] + [g.shape[d] * (k + 1) // n - 3 * (k == 0) for k in range(n - 1)] + [g.shape[d]]
        return g.narrow(d, cut[r], cut[r + 1] - cut[r])

    ranks = Ranks(n)
    outs = ranks.run(lambda r, reduce: orthogonalize([parts(g, d, r) for g, d in zip(gs, splits)], split=splits, all_reduce=reduce))
    assert len(set(ranks.calls)) == 1 and ranks.calls[0] == 1 + 5
    for i, (g, d) in enumerate(zip(gs, splits)):
        got = outs[0][i] if d is None else torch.cat([o[i] for o in outs], d)
        near(got, exact(g), what=str(i))


def test_failing_reduce():
    def fails(t):
        raise ZeroDivisionError("the network is down")
    with pytest.raises(ZeroDivisionError, match="the network is down"):
        orthogonalize([draw((8, 8))], split=[0], all_reduce=fails)
    near(orthogonalize([draw((8, 8))], split=[0], all_reduce=lambda t: None)[0], exact(draw((8, 8))))


# ------------------------------------------------------------------- Muon

FIELDS = {"f32": (F32, None, F32, F32), "mixed": (BF16, F32, F32, BF16), "bf16": (BF16, None, BF16, BF16),
          "mixed moments": (BF16, F32, BF16, F32)}       # param, master, exp_avg, gradients
MU, LR, DECAY = 0.9, 0.02, 0.3


def share(fields, shapes):
    pt, mt, at, _ = FIELDS[fields]
    state = {}
    for i, s in enumerate(shapes):
        w = draw(s, seed=100 + i, std=0.05)
        e = {"param": w.to(pt), "exp_avg": draw(s, seed=200 + i, std=0.01).to(at)}
        if mt:
            e["master"] = w.clone()
        state[f"p{i}"] = e
    return state


def muon64(w, m, g, nesterov=True, scale=1.0, factor=1.0, moment=F32):
    """The momentum and the weight in 64 bits, and how far they may be off; the weight goes by the momentum that is stored."""
    g = factor * g.double()
    m64 = MU * m.double() + (1 - MU) * g
    off_m = 3 * u * (MU * m.double().abs() + (1 - MU) * g.abs())
    off_m = off_m + U[moment] * (m64.abs() + off_m) + 2.0 ** -133
    return m64, off_m


def stepped(w, m_new, g, nesterov, scale, factor=1.0):
    g = factor * g.double()
    m = m_new.double()
    x = exact(MU * m + (1 - MU) * g if nesterov else m)
    want = w.double() * (1 - LR * DECAY) - LR * scale * x
    return want, x


SHARE = [(24, 16), (16, 8), (130, 64), (64, 200), (300, 300), (1, 7)]


@pytest.mark.parametrize("fields", FIELDS)
@pytest.mark.parametrize("nesterov", [True, False])
def test_step(fields, nesterov):
    state = share(fields, SHARE)
    gt = FIELDS[fields][3]
    grads = {n: draw(tuple(e["param"].shape), seed=300 + i, std=0.02, dtype=gt) for i, (n, e) in enumerate(state.items())}
    before = {n: {f: t.clone() for f, t in e.items()} for n, e in state.items()}
    optimizer = ShardMuon(state, lr=LR, momentum=MU, nesterov=nesterov, weight_decay=DECAY)
    versions = [t._version for e in state.values() for t in e.values()]
    assert optimizer.step(grads) is None
    assert all(t._version > v for t, v in zip((t for e in state.values() for t in e.values()), versions))
    for n, e in state.items():
        b = before[n]
        key = "master" if "master" in b else "param"
        r, c = e["param"].shape
        m64, off_m = muon64(b[key], b["exp_avg"], grads[n], moment=e["exp_avg"].dtype)
        assert bool(((e["exp_avg"].double() - m64).abs() <= off_m).all()), n
        scale = math.sqrt(max(1.0, r / c))
        want, x = stepped(b[key], e["exp_avg"], grads[n], nesterov, scale)
        off = float((e[key].double() - want).norm())
        allowed = LR * scale * (growth(5) + 4 * u) * float(x.norm()) + (4 * u + U[e[key].dtype]) * float(want.norm() + b[key].double().norm())
        assert off <= allowed, (n, off, allowed)
        if key == "master":
            assert torch.equal(e["param"], e["master"].to(BF16)), n
    assert optimizer.state() is state


def test_same_as_its_parts():
    """A step is the momentum, orthogonalize and the update: with steps of 1, missing gradients and other rates."""
    state = share("f32", SHARE)
    before = {n: {f: t.clone() for f, t in e.items()} for n, e in state.items()}
    grads = [None if i == 2 else draw(s, seed=i) for i, s in enumerate(SHARE)]
    optimizer = ShardMuon(state, lr=LR, momentum=MU, nesterov=False, weight_decay=0.0, adjust_lr="match_rms_adamw")
    optimizer.step(grads)
    for i, (n, e) in enumerate(state.items()):
        if i == 2:
            assert all(torch.equal(t, before[n][f]) for f, t in e.items())
            continue
        x, = orthogonalize([e["exp_avg"]])
        want = before[n]["param"].double() - LR * 0.2 * math.sqrt(max(e["param"].shape)) * x.double()
        size = float(x.double().norm()) * LR * 0.2 * math.sqrt(max(e["param"].shape))
        assert float((e["param"].double() - want).norm()) <= growth(5) * size + 4 * u * float(want.norm())
    optimizer.lr = 0.0
    kept = {n: e["param"].clone() for n, e in state.items()}
    optimizer.step(grads)
    assert all(torch.equal(e["param"], kept[n]) for n, e in state.items())


def test_clipped():
    grads = [draw(s, seed=i) for i, s in enumerate(SHARE)]
    q = grad_square_sum(grads)
    results = []
    for kw in (dict(max_norm=1.0), dict(max_norm=1.0, square_sum=q), None):
        state = share("f32", SHARE)
        optimizer = ShardMuon(state, lr=LR, momentum=MU)
        if kw is None:
            norm = math.sqrt(float(q))
            optimizer.step([g * min(1.0, 1.0 / (norm + 1e-6)) for g in grads])
        else:
            norm = optimizer.step(grads, **kw)
            assert torch.equal(norm, grad_norm(grads))
        results.append(state)
    for n in results[0]:
        for f in ("param", "exp_avg"):
            assert torch.equal(results[0][n][f], results[1][n][f])
            # the factor is rounded once more
            torch.testing.assert_close(results[0][n][f], results[2][n][f], rtol=1e-4, atol=1e-6)
    assert torch.equal(grads[0], draw(SHARE[0], seed=0))


def test_split_share():
    """Two ranks' halves of a share make the step of the whole one."""
    from suika_amd import ParamLayout, TensorMeta, split_matrices
    cut = {"gate": 0, "down": 1, "whole": None}
    shapes = {"gate": (96, 64), "down": (64, 96), "whole": (32, 64)}

    def layout(tp):
        return ParamLayout.from_metas({r: {n: TensorMeta(name=n, dtype=BF16, shape=shapes[n],
                                                         tp_meta=None if cut[n] is None or tp == 1 else (cut[n], r, tp))
                                           for n in shapes} for r in range(tp)})

    def part(t, n, r, tp):
        return (t if cut[n] is None or tp == 1 else t.chunk(tp, cut[n])[r]).contiguous().clone()

    whole = dict(zip(shapes, share("mixed", list(shapes.values())).values()))
    grads = {n: draw(s, seed=40 + i, dtype=BF16) for i, (n, s) in enumerate(shapes.items())}
    parts = [{n: {f: part(t, n, r, 2) for f, t in e.items()} for n, e in whole.items()} for r in range(2)]
    ShardMuon(whole, lr=LR, momentum=MU, splits=split_matrices(layout(1), 0)).step(grads)

    def one(r, reduce):
        o = ShardMuon(parts[r], lr=LR, momentum=MU, splits=split_matrices(layout(2), r), all_reduce=reduce)
        o.step({n: part(g, n, r, 2) for n, g in grads.items()})

    Ranks(2).run(one)
    for n in shapes:
        for f in ("exp_avg", "master"):
            got = parts[0][n][f] if cut[n] is None else torch.cat([p[n][f] for p in parts], cut[n])
            if f == "exp_avg":
                assert torch.equal(got, whole[n][f])
            else:
                r, c = shapes[n]
                off = 2 * growth(5) * LR * math.sqrt(max(1.0, r / c)) * math.sqrt(min(r, c)) * 1.2 + 4 * u * float(got.norm())
                assert float((got - whole[n][f]).norm()) <= off, n


def test_captured_step():
    state = share("mixed", SHARE)
    other = {n: {f: t.clone() for f, t in e.items()} for n, e in state.items()}
    grads = [draw(s, dtype=BF16) for s in SHARE]
    eager, kept = ShardMuon(other, lr=LR), ShardMuon(state, lr=LR)
    ShardMuon(share("mixed", SHARE), lr=LR).step(grads, max_norm=1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = kept.step(grads, max_norm=1.0)
    for k in range(3):
        for i, g in enumerate(grads):
            g.copy_(draw(SHARE[i], seed=50 * k + i))
        want = eager.step(grads, max_norm=1.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want)
        assert all(torch.equal(state[n][f], other[n][f]) for n in state for f in state[n])


def test_refused_steps_change_nothing():
    state = share("f32", SHARE)
    before = {n: {f: t.clone() for f, t in e.items()} for n, e in state.items()}
    optimizer = ShardMuon(state)
    grads = [draw(s) for s in SHARE]
    for bad, word in [(grads[:-1], "tensors for a state"), ([g.t() for g in grads], "dense tensor"), ([g.half() for g in grads], "dtype"),
                      ([g.cpu() for g in grads], "dense tensor"), ({"nobody": grads[0]}, "unknown"),
                      ([next(iter(state.values()))["param"]] + grads[1:], "overlap")]:
        with pytest.raises(PlanError, match=word):
            optimizer.step(bad)
    for kw, word in [(dict(max_norm=-1.0), "max_norm"), (dict(square_sum=grad_square_sum(grads)), "without max_norm")]:
        with pytest.raises(PlanError, match=word):
            optimizer.step(grads, **kw)
    optimizer.lr = -1.0
    with pytest.raises(PlanError, match="lr"):
        optimizer.step(grads, max_norm=1.0)
    optimizer.lr = 1.0
    first = next(iter(state.values()))
    first["param"].data = torch.zeros(16, 24, device=DEV)
    first["exp_avg"].data = torch.zeros(16, 24, device=DEV)
    with pytest.raises(PlanError, match="another shape"):
        optimizer.step([draw((16, 24))] + grads[1:])
    assert all(torch.equal(t, before[n][f]) for n, e in list(state.items())[1:] for f, t in e.items())
    with pytest.raises(PlanError, match="a matrix"):
        ShardMuon({"b": {"param": torch.zeros(3, device=DEV), "exp_avg": torch.zeros(3, device=DEV)}})


def test_matrices_from_an_iterator():
    gs = [draw((20, 30)), draw((70, 90))]
    want = orthogonalize(gs)
    for mode in (torch.enable_grad, torch.no_grad):
        with mode():
            for given in (iter(gs), (g for g in gs), torch.stack([gs[0], gs[0]])):
                got = orthogonalize(given)
                assert len(got) == 2 and torch.equal(got[0], want[0])


def test_outputs_that_want_a_gradient():
    import torch.autograd.forward_ad as fwd
    g, out = draw((8, 8)), draw((8, 8), seed=1).requires_grad_()
    before = out.detach().clone()
    with pytest.raises(PlanError, match="out: one wants a gradient"):
        orthogonalize([g], out=[out])
    with fwd.dual_level():
        with pytest.raises(PlanError, match="forward-mode"):
            orthogonalize([g], out=[fwd.make_dual(before.clone(), g)])
    assert torch.equal(out, before)
    with torch.no_grad():
        orthogonalize([g], out=iter([out]))
    assert torch.equal(out.detach(), orthogonalize([g])[0])


def test_a_local_norm_does_not_clip_parts():
    """Ranks would clip the parts of one matrix by factors of their own, whose Gram matrices do not add up to its own."""
    shapes = {"cut": (16, 24), "whole": (70, 90)}
    state = dict(zip(shapes, share("f32", list(shapes.values())).values()))
    before = {n: {f: t.clone() for f, t in e.items()} for n, e in state.items()}
    grads = {n: draw(s, seed=i) for i, (n, s) in enumerate(shapes.items())}
    optimizer = ShardMuon(state, lr=LR, momentum=MU, splits={"cut": (0, 32)}, all_reduce=lambda t: None)
    with pytest.raises(PlanError, match="square_sum"):
        optimizer.step(grads, max_norm=1.0)
    assert all(torch.equal(t, before[n][f]) for n, e in state.items() for f, t in e.items())
    # of whole matrices alone it is theirs, and a sum over the ranks serves all
    assert torch.equal(optimizer.step({"whole": grads["whole"]}, max_norm=1.0), grad_norm([grads["whole"]]))
    q = grad_square_sum(list(grads.values()))
    assert torch.equal(optimizer.step(grads, max_norm=1.0, square_sum=q), grad_norm(list(grads.values())))


@pytest.mark.parametrize("fails_at", [0, 1, 5, 6, 9])
def test_failing_reduce_of_a_step(fails_at):
    """More cut matrices than go through the steps together (48, with a call for their norms and one each step), whole
    and small ones: all moments are updated, the weights of uncut matrices too, and of cut ones all or none of a weight."""
    shapes = [(8, 12)] * 50 + [(70, 90), (20, 16)]
    state = share("mixed", shapes)
    names = list(state)
    grads = [draw(s, seed=300 + i, dtype=BF16) for i, s in enumerate(shapes)]
    other = {n: {f: t.clone() for f, t in e.items()} for n, e in state.items()}
    before = {n: e["master"].clone() for n, e in state.items()}
    splits = {n: (0, 8) for n in names[:50]}
    calls = []

    def fails(t):
        calls.append(t)
        if len(calls) == fails_at + 1:
            raise ZeroDivisionError("the network is down")

    ShardMuon(other, lr=LR, momentum=MU, splits=splits, all_reduce=lambda t: None).step(grads)
    with pytest.raises(ZeroDivisionError, match="the network is down"):
        ShardMuon(state, lr=LR, momentum=MU, splits=splits, all_reduce=fails).step(grads)
    assert len(calls) == fails_at + 1
    stepped = {n for n in names if not torch.equal(state[n]["master"], before[n])}
    assert stepped == set(names[50:]) | (set(names[:48]) if fails_at > 5 else set())
    for n, e in state.items():
        assert torch.equal(e["exp_avg"], other[n]["exp_avg"]), n
        if n in stepped:
            assert torch.equal(e["master"], other[n]["master"]) and torch.equal(e["param"], other[n]["param"]), n



# --------------------------------------------------- products of large tiles

# One matrix of 16 x 16 tiles of 256, with odd remainders: X goes through its steps in these,
# and from 32 tiles of 128 a side on so do A and B.
LARGE = [(3843, 3901), (3903, 3842), (4003, 4069), (4071, 4001)]


def kernels_of(f):
    """The kernels that a call launches."""
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as p:
        f()
        torch.cuda.synchronize()
    return {e.key for e in p.key_averages()}


def iterates(g, steps=5):
    """The result in 64 bits, and the norms of the iterates after each step."""
    x = g.double()
    x = x / x.norm()
    flip = x.shape[0] > x.shape[1]
    x = (x.t() if flip else x).contiguous()
    a, b, c = COEFFICIENTS
    sizes = []
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
        sizes.append(float(x.norm()))
    return (x.t() if flip else x), sizes


def near_everywhere(got, want, sizes, what=""):
    """A step's roundings are 4 * 2^-22 of its result's size and grow by 3.4445 in each later one: together the bound on
    the norm of all.  Rows, columns and elements of a normal matrix are alike, so no row's or column's share of that is
    more than 4 times its part, and no element's more than 16 times the root of the mean square."""
    dt, n = got.dtype, len(sizes)
    bound = sum(4 * 2.0 ** -22 * s * COEFFICIENTS[0] ** (n - 1 - j) for j, s in enumerate(sizes))
    off = got.double() - want
    assert float(off.norm()) <= bound + U[dt] * float(want.norm()), f"{what}: {float(off.norm()):.2e}, {bound:.2e} allowed"
    for d in (0, 1):
        allowed = 4 * bound / math.sqrt(want.shape[1 - d]) + U[dt] * want.norm(dim=d)
        assert bool((off.norm(dim=d) <= allowed).all()), f"{what}: along {d}"
    assert bool((off.abs() <= 16 * bound / math.sqrt(want.numel()) + U[dt] * want.abs()).all()), f"{what}: an element"


@pytest.mark.parametrize("shape", LARGE, ids=str)
def test_large_tiles(shape):
    g = draw(shape)
    want, sizes = iterates(g)
    for dtype in (F32, BF16):
        out = torch.empty(shape[0], shape[1] + 3, dtype=dtype, device=DEV)[:, 1:-2]
        names = kernels_of(lambda: orthogonalize([g], out=[out]))
        wanted = ["update_kernel<256>", "last_kernel<256>"]
        if min(shape) > 31 * 128:
            wanted += ["symmetric_kernel<256, false>", "symmetric_kernel<256, true>"]
        assert all(any(k in n for n in names) for k in wanted), sorted(n for n in names if "kernel<" in n)
        near_everywhere(out, want, sizes, str(dtype))
    # as a part of itself, whose Gram matrices go to the host program
    for split in (0, 1):
        got, = orthogonalize([g], split=[split], all_reduce=lambda t: None)
        near_everywhere(got, want, sizes, f"split {split}")


@pytest.mark.parametrize("shape", LARGE, ids=str)
@pytest.mark.parametrize("fields", ["mixed", "bf16"])
def test_large_tiles_of_weights(shape, fields):
    state = share(fields, [shape])
    entry = state["p0"]
    key = "master" if "master" in entry else "param"
    old = {f: t.clone() for f, t in entry.items()}
    grad = draw(shape, seed=300, std=0.02, dtype=FIELDS[fields][3])
    optimizer = ShardMuon(state, lr=LR, momentum=MU, weight_decay=DECAY, adjust_lr="none")
    assert any("last_kernel<256>" in n for n in kernels_of(lambda: optimizer.step([grad])))
    m64, off_m = muon64(old[key], old["exp_avg"], grad, moment=entry["exp_avg"].dtype)
    assert bool(((entry["exp_avg"].double() - m64).abs() <= off_m).all())
    x, sizes = iterates(MU * entry["exp_avg"].double() + (1 - MU) * grad.double())
    want = old[key].double() * (1 - LR * DECAY) - LR * x
    bound = LR * sum(4 * 2.0 ** -22 * s * COEFFICIENTS[0] ** (4 - j) for j, s in enumerate(sizes))
    # the decay factor, the two products and the difference, and what is stored
    off = (entry[key].double() - want).abs()
    allowed = 16 * bound / math.sqrt(want.numel()) + 2 * u * (old[key].double().abs() + LR * x.abs()) + U[entry[key].dtype] * want.abs()
    assert bool((off <= allowed + 2.0 ** -133).all())
    if key == "master":
        assert torch.equal(entry["param"], entry["master"].to(BF16))


@pytest.mark.parametrize("shape", [(65, 64), (127, 130), (129, 257), (300, 299), (520, 530), (200, 1000), (1000, 200)], ids=str)
def test_every_element(shape):
    g = draw(shape)
    want, sizes = iterates(g)
    near_everywhere(orthogonalize([g])[0], want, sizes)


# --------------------------------------------------------- torch.optim.Muon

@pytest.mark.parametrize("adjust", ["original", "match_rms_adamw"])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shape", [(96, 40), (40, 96)], ids=str)
def test_steps_of_torch(shape, nesterov, adjust):
    """Two steps beside torch.optim.Muon, whose one Newton-Schulz step is in bf16: X, A, A A, B, B X and the sum rounded
    to 2^-8, each of at most |a| + |b| + |c| of X's norm of 1.  Its momentum is in 32 bits, as here."""
    lr, decay = 0.1, 0.5
    w = draw(shape, seed=1, std=0.5)
    theirs = torch.nn.Parameter(w.clone())
    torch_muon = torch.optim.Muon([theirs], lr=lr, weight_decay=decay, momentum=MU, nesterov=nesterov, ns_steps=1,
                                  adjust_lr_fn=adjust)
    state = {"w": {"param": w.clone(), "exp_avg": torch.zeros_like(w)}}
    ours = ShardMuon(state, lr=lr, weight_decay=decay, momentum=MU, nesterov=nesterov, ns_steps=1, adjust_lr=adjust)
    rate = lr * (math.sqrt(max(1.0, shape[0] / shape[1])) if adjust == "original" else 0.2 * math.sqrt(max(shape)))
    for k in range(1, 3):
        theirs.grad = draw(shape, seed=10 + k, std=0.02)
        ours.step([theirs.grad])
        torch_muon.step()
        m = torch_muon.state[theirs]["momentum_buffer"]
        assert bool(((state["w"]["exp_avg"] - m).abs() <= 8 * u * (m.abs() + theirs.grad.abs())).all())
        allowed = k * (rate * 6 * U[BF16] * sum(map(abs, COEFFICIENTS)) + 8 * u * float(w.norm()))
        assert float((state["w"]["param"] - theirs.detach()).norm()) <= allowed
    # without the decay, or at the other rate, the weights would be farther away than that
    assert 2 * lr * decay * float(w.norm()) > 4 * allowed
