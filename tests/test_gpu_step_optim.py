"""Gradient norm, clipping and AdamW on the GPU against the formulas in 64 bits.

The bounds come from the kernels' roundings.  u = 2^-24 is half a unit in the
last place of a float32, U(type) of the stored type.  A sum of squares is
formed in 64 bits, so a norm is one float32 rounding away: 2u.  A clipped
element is rounded as factor, as product and where it is stored: 3u + U.
"""
import math

import pytest
import torch

from suika_amd import PlanError, ShardAdamW, clip_grads, grad_norm, grad_square_sum

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {t: torch.finfo(t).eps / 2 for t in (F32, BF16, F16)}
u = U[F32]
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -25}     # below the smallest value that keeps its bits
DEV = "cuda"


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def randn(g, n, dtype=F32, std=1.0, shift=0):
    """n elements that start ``shift`` elements into an allocation."""
    t = torch.empty(n + shift, device=DEV, dtype=dtype)[shift:]
    t.copy_(torch.randn(n, generator=g, device=DEV) * std)
    return t


def square_sum64(grads):
    return sum(float(t.double().square().sum()) for t in grads if t is not None)


LENGTHS = [[], [0], [1], [7], [0, 3, 0, 1], [255, 256, 257], [16383], [16384], [16385], [2 ** 20 + 13],
           [5] * 189, [5] * 190, [64, 1] * 200, [32768], [32769], [40000] * 190, [100003, 17, 2 ** 18, 0, 31]]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: f"{len(v)}x{max(v, default=0)}")
def test_norm(lengths, shift, dtype):
    g = gen(1)
    grads = [randn(g, n, dtype, 1e-3, shift) for n in lengths]
    want = square_sum64(grads)
    got, q = grad_norm(grads), grad_square_sum(grads)
    assert got.dtype == F32 and got.shape == () and q.dtype == torch.float64 and q.shape == ()
    assert abs(float(q) - want) <= 1e-13 * want
    assert abs(float(got) - math.sqrt(want)) <= 2 * u * math.sqrt(want)
    assert torch.equal(grad_square_sum(grads), q)


def test_norm_mixed_types_shapes_and_none():
    g = gen(2)
    grads = [randn(g, 1000).view(10, 100), None, randn(g, 513, BF16), randn(g, 77, F16), randn(g, 1).view(())]
    want = math.sqrt(square_sum64(grads))
    assert abs(float(grad_norm(grads)) - want) <= 2 * u * want
    assert float(grad_norm(tuple(grads))) == float(grad_norm(grads))
    assert float(grad_norm([None])) == 0.0


def test_norm_of_large_and_small_values():
    big = torch.full((1000,), 3e38, device=DEV)
    small = torch.full((1000,), 1e-30, device=DEV)
    assert math.isclose(float(grad_square_sum([big])), 1000 * float(big[0]) ** 2, rel_tol=1e-13)
    assert math.isclose(float(grad_norm([small])), math.sqrt(1000) * float(small[0]), rel_tol=2 * u)
    assert math.isinf(float(grad_norm([big])))        # the norm itself is beyond float32
    big[7] = math.inf
    assert math.isinf(float(grad_norm([big])))
    big[8] = math.nan
    assert math.isnan(float(grad_norm([big])))


CLIP_TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, BF16), (F16, F32)]


def clipped64(t, norm, max_norm):
    return t.double() * min(1.0, max_norm / (norm + 1e-6))


def assert_clipped(got, want):
    dt = got.dtype
    off = (got.double() - want).abs()
    assert bool((off <= (3 * u + U[dt]) * want.abs() + TINY[dt]).all()), float(off.max())


@pytest.mark.parametrize("src,dst", CLIP_TYPES)
@pytest.mark.parametrize("lengths", [[1], [4095, 4096, 4097], [5] * 130, [100003, 0, 17]],
                         ids=lambda v: f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("shift", [0, 1])
def test_clip_out_of_place(src, dst, lengths, shift):
    g = gen(3)
    grads = [randn(g, n, src, 0.5, shift) for n in lengths]
    outs = [torch.full((n + 2,), 9.0, device=DEV, dtype=dst) for n in lengths]
    inner = [o[1:-1] for o in outs]
    norm = math.sqrt(square_sum64(grads))
    before = [t.clone() for t in grads]
    got = clip_grads(grads, 0.3 * norm, out=inner)
    assert abs(float(got) - norm) <= 2 * u * norm
    for t, b, o, whole in zip(grads, before, inner, outs):
        assert torch.equal(t, b)
        assert_clipped(o, clipped64(t, norm, 0.3 * norm))
        assert float(whole[0]) == 9.0 and float(whole[-1]) == 9.0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_clip_in_place(dtype):
    g = gen(4)
    grads = [randn(g, n, dtype, 0.5).view(-1, 1) for n in (4097, 3, 0, 70000)]
    norm = math.sqrt(square_sum64(grads))
    before = [t.clone() for t in grads]
    versions = [t._version for t in grads]
    assert abs(float(clip_grads(grads, 2 * norm)) - norm) <= 2 * u * norm
    assert all(torch.equal(t, b) for t, b in zip(grads, before))          # nothing to clip
    clip_grads(grads, 0.1 * norm)
    for t, b in zip(grads, before):
        assert_clipped(t, clipped64(b, norm, 0.1 * norm))
    assert all(t._version > v for t, v in zip(grads, versions))


def test_clip_by_another_ranks_sum():
    g = gen(5)
    grads = [randn(g, 1000), None]
    q = grad_square_sum(grads) * 4
    before = grads[0].clone()
    norm = clip_grads(grads, 1.0, square_sum=q)
    want = math.sqrt(square_sum64([before]) * 4)
    assert abs(float(norm) - want) <= 2 * u * want
    assert_clipped(grads[0], clipped64(before, want, 1.0))
    assert float(clip_grads([], 1.0, square_sum=q)) == float(norm)
    assert float(clip_grads([None], 1.0)) == 0.0


def test_clip_infinite_and_nan():
    t = torch.ones(5000, device=DEV)
    t[10] = math.inf
    clip_grads([t], 1.0)
    assert bool(t[10].isnan()) and float(t[11]) == 0.0
    t = torch.ones(5000, device=DEV)
    t[10] = math.nan
    clip_grads([t], 1.0)
    assert bool(t.isnan().all())


# ------------------------------------------------------------------ AdamW

def make_state(g, lengths, fields, shift=0):
    state = {}
    for i, n in enumerate(lengths):
        w = randn(g, n, std=0.02, shift=shift)
        moment = BF16 if fields == "bf16" else F32
        v = randn(g, n, std=1e-6, shift=shift).abs_()
        entry = {"param": w if fields == "f32" else w.to(BF16), "exp_avg": randn(g, n, moment, 1e-3, shift),
                 "exp_avg_sq": v.to(moment), "step": torch.tensor(6.0)}
        if fields == "master":
            entry["master"] = w
        state[f"p{i}"] = entry
    return state


def adamw64(entry, grad, factor, t, lr, betas, eps, decay):
    """New fields in 64 bits and how far the kernel's may be from them."""
    f = {k: v.double() for k, v in entry.items() if k != "step"}
    b1, b2 = betas
    g = grad.double() * factor
    m = b1 * f["exp_avg"] + (1 - b1) * g
    v = b2 * f["exp_avg_sq"] + (1 - b2) * g * g
    # factors of one rounding each (beta, 1 - beta, clip factor), the products and the sum
    m_off = 6 * u * (b1 * f["exp_avg"].abs() + (1 - b1) * g.abs()) + 2.0 ** -149
    v_off = 8 * u * v + 2.0 ** -148
    w = f.get("master", f["param"])
    root = (v / (1 - b2 ** t)).sqrt() + eps
    change = lr / (1 - b1 ** t) * m / root
    # the root of a sum off by 8u is off by 4u, its scale, sum, quotient and product by one each
    change_off = 12 * u * change.abs() + lr / (1 - b1 ** t) * m_off / root
    small = (v < 1e-37).double()          # v itself is below what float32 keeps with all bits
    change_off = change_off + small * change.abs()
    new = w * (1 - lr * decay) - change
    w_off = 2 * u * w.abs() + u * new.abs() + change_off
    return {"w": (new, w_off), "exp_avg": (m, m_off), "exp_avg_sq": (v, v_off)}


def assert_near(got, want, off, what):
    dt = got.dtype
    allowed = off + (U[dt] * (want.abs() + off) + TINY[dt] if dt != F32 else 0)
    diff = (got.double() - want).abs()
    assert bool((diff <= allowed).all()), (what, float(diff.max()), float((diff / allowed).max()))


def check_step(state, old, grads, opt, max_norm, norm):
    factor = 1.0 if max_norm is None else min(1.0, max_norm / (norm + 1e-6))
    for (name, entry), grad in zip(state.items(), grads):
        if grad is None:
            assert all(torch.equal(entry[f], old[name][f]) for f in entry)
            continue
        want = adamw64(old[name], grad, factor, opt.steps, opt.lr, opt.betas, opt.eps, opt.weight_decay)
        assert_near(entry["exp_avg"], *want["exp_avg"], name)
        assert_near(entry["exp_avg_sq"], *want["exp_avg_sq"], name)
        if "master" in entry:
            assert_near(entry["master"], *want["w"], name)
            assert torch.equal(entry["param"], entry["master"].to(BF16))
        else:
            assert_near(entry["param"], *want["w"], name)


def copy_of(state):
    return {n: {f: t.clone() for f, t in e.items()} for n, e in state.items()}


@pytest.mark.parametrize("fields,grad", [("f32", F32), ("f32", BF16), ("master", BF16), ("master", F32),
                                         ("bf16", BF16), ("bf16", F32)])
@pytest.mark.parametrize("lengths", [[1], [0, 3], [2047, 2048, 2049], [7] * 203, [100003, 1, 4096]],
                         ids=lambda v: f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("max_norm", [None, 0.01])
def test_adamw_step(fields, grad, lengths, shift, max_norm):
    g = gen(6)
    state = make_state(g, lengths, fields, shift)
    grads = [randn(g, n, grad, 1e-3, shift) for n in lengths]
    old = copy_of(state)
    kept = [t.clone() for t in grads]
    opt = ShardAdamW(state, lr=2e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    assert opt.steps == 6
    got = opt.step(grads, max_norm=max_norm)
    norm = math.sqrt(square_sum64(grads))
    if max_norm is None:
        assert got is None
    else:
        assert abs(float(got) - norm) <= 2 * u * norm
    assert opt.steps == 7
    check_step(state, old, grads, opt, max_norm, norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, kept))
    assert all(float(e["step"]) == 7 for e in opt.state().values())


def test_adamw_against_torch_over_steps():
    """Ten steps next to torch.optim.AdamW in 64 bits: the weights stay within
    what ten steps' roundings allow (each step's are below 16u of the weight
    and of its change, and a moment's relative error is at most that times
    the steps it remembers)."""
    g = gen(7)
    lengths = [1000, 33]
    state = {f"p{i}": {"param": randn(g, n, std=0.02), "exp_avg": torch.zeros(n, device=DEV),
                       "exp_avg_sq": torch.zeros(n, device=DEV)} for i, n in enumerate(lengths)}
    twins = [torch.nn.Parameter(e["param"].double()) for e in state.values()]
    opt = ShardAdamW(state, lr=1e-2, weight_decay=0.05)
    ref = torch.optim.AdamW(twins, lr=1e-2, weight_decay=0.05, betas=(0.9, 0.999), eps=1e-8)
    for k in range(10):
        grads = {n: randn(g, e["param"].numel()) for n, e in state.items()}
        for t, gr in zip(twins, grads.values()):
            t.grad = gr.double()
        opt.step(grads)
        ref.step()
    for t, e in zip(twins, state.values()):
        off = (e["param"].double() - t.detach()).abs()
        assert bool((off <= 10 * 16 * u * (t.detach().abs() + 10 * 1e-2 * 4)).all()), float(off.max())
    assert opt.steps == 10 and float(opt.state()["p0"]["step"]) == 10


def test_adamw_special_values():
    """Zeros stay put, an infinite gradient makes NaN where it is, as the
    formula does, and its neighbours go on."""
    state = {"w": {"param": torch.zeros(2050, device=DEV), "exp_avg": torch.zeros(2050, device=DEV),
                   "exp_avg_sq": torch.zeros(2050, device=DEV)}}
    opt = ShardAdamW(state, lr=1.0, weight_decay=0.5)
    grad = torch.zeros(2050, device=DEV)
    opt.step([grad])
    assert not bool(state["w"]["param"].any())
    grad[5] = math.inf
    grad[2049] = math.nan
    grad[6] = 1.0
    opt.step([grad])
    p = state["w"]["param"]
    assert bool(p[5].isnan()) and bool(p[2049].isnan()) and float(p[6]) < 0 and not bool(p[7:2049].any())


def test_adamw_missing_gradients_and_sum_of_other_ranks():
    g = gen(8)
    state = make_state(g, [100, 200, 300], "master")
    old = copy_of(state)
    grads = [randn(g, 100), None, randn(g, 300)]
    opt = ShardAdamW(state)
    q = grad_square_sum(grads) * 9
    got = opt.step({"p0": grads[0], "p2": grads[2]}, max_norm=1.0, square_sum=q)
    norm = math.sqrt(square_sum64(grads) * 9)
    assert abs(float(got) - norm) <= 2 * u * norm
    check_step(state, old, grads, opt, 1.0, norm)


def test_adamw_refusals():
    g = gen(9)
    state = make_state(g, [64, 8], "master")
    opt = ShardAdamW(state)
    good = [randn(g, 64), randn(g, 8)]
    before = copy_of(state)
    for grads, match in [([good[0]], "1 tensors for a state of 2"),
                         ([good[0], randn(g, 7)], "like the weight"),
                         ([good[0], good[1].cpu()], "like the weight"),
                         ([good[0].half(), good[1]], "Half"),
                         ([randn(g, 128)[::2], good[1]], "like the weight"),
                         ({"p0": good[0], "other": good[1]}, "unknown"),
                         ([state["p0"]["master"], good[1]], "overlaps")]:
        with pytest.raises(PlanError, match=match):
            opt.step(grads)
    with pytest.raises(PlanError, match="square_sum"):
        opt.step(good, max_norm=1.0, square_sum=torch.ones((), device=DEV))
    with pytest.raises(PlanError, match="without max_norm"):
        opt.step(good, square_sum=torch.ones((), device=DEV, dtype=torch.float64))
    with pytest.raises(PlanError, match="max_norm"):
        opt.step(good, max_norm=-1.0)
    opt.lr = -1.0
    with pytest.raises(PlanError, match="lr"):
        opt.step(good)
    assert opt.steps == 6
    assert all(torch.equal(state[n][f], before[n][f]) for n in state for f in state[n])
    half = {"w": {"param": good[0].half(), "exp_avg": good[0].clone(), "exp_avg_sq": good[0].clone()}}
    with pytest.raises(PlanError, match="weight of dtype"):
        ShardAdamW(half)
    with pytest.raises(PlanError, match="different shapes"):
        ShardAdamW({"w": {"param": good[0], "exp_avg": good[1], "exp_avg_sq": good[1].clone()}})
    with pytest.raises(PlanError, match="moments"):
        ShardAdamW({"w": {"param": good[0], "exp_avg": good[0].clone(), "exp_avg_sq": good[0].bfloat16()}})
    with pytest.raises(PlanError, match="master"):
        ShardAdamW({"w": {"param": good[0].clone(), "master": good[0], "exp_avg": good[0].clone(),
                          "exp_avg_sq": good[0].clone()}})


def test_norm_and_clip_refusals():
    t = torch.ones(8, device=DEV)
    for bad, match in [([t.double()], "Double"), ([t.cpu()], "cpu"), ([t[::2]], "contiguous"), ([3], "not a tensor")]:
        with pytest.raises(PlanError, match=match):
            grad_norm(bad)
        with pytest.raises(PlanError, match=match):
            clip_grads(bad, 1.0)
    with pytest.raises(PlanError, match="max_norm"):
        clip_grads([t], -1.0)
    with pytest.raises(PlanError, match="2 tensors"):
        clip_grads([t], 1.0, out=[t, t])
    with pytest.raises(PlanError, match="shape"):
        clip_grads([t], 1.0, out=[torch.ones(2, 4, device=DEV)])
    with pytest.raises(PlanError, match="overlaps"):
        clip_grads([t, t], 1.0)
    assert bool((t == 1).all())


def test_on_another_stream_and_in_a_graph():
    g = gen(10)
    grads = [randn(g, n, BF16) for n in (5000, 3, 70001)]
    outs = [torch.empty_like(t, dtype=F32) for t in grads]
    want = grad_norm(grads)
    clip_grads(grads, 1.0, out=outs)
    expect = [o.clone() for o in outs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for o in outs:
            o.zero_()
        norm = clip_grads(grads, 1.0, out=outs)
        graph = torch.cuda.CUDAGraph()
    side.synchronize()
    assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(outs, expect))
    with torch.cuda.graph(graph, stream=side):
        norm = clip_grads(grads, 1.0, out=outs)
    for k in range(3):
        scaled = [t * (k + 1) for t in grads]
        for t, s in zip(grads, scaled):
            t.copy_(s)
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        again = [torch.empty_like(o) for o in outs]
        eager = clip_grads(grads, 1.0, out=again)
        assert torch.equal(norm, eager) and all(torch.equal(a, b) for a, b in zip(outs, again))


def test_adamw_refuses_a_capture():
    state = make_state(gen(11), [64], "f32")
    opt = ShardAdamW(state)
    grad = [torch.ones(64, device=DEV)]
    opt.step(grad)
    before = copy_of(state)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(PlanError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step(grad)
    torch.cuda.synchronize()
    assert opt.steps == 7 and all(torch.equal(state["p0"][f], before["p0"][f]) for f in before["p0"])
