"""Every parameter of ShardAdamW counts its own updates, as torch.optim.AdamW
does: gradients that are missing for a while, states whose steps differ, and
names of one tensor.

Against torch's AdamW in 64 bits over K steps: each step's roundings are below
16u of the weight and of its change, which is at most 4 lr here, and a moment's
relative error is at most that times the steps it remembers; so the weights
stay within K 16 u (|w| + K lr 4), u = 2^-24."""
import pytest
import torch

from suika_amd import PlanError, ShardAdamW

pytestmark = pytest.mark.gpu
DEV = "cuda"
u = 2.0 ** -24


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def fresh(g, lengths):
    return {f"p{i}": {"param": torch.randn(n, generator=g, device=DEV) * 0.02, "exp_avg": torch.zeros(n, device=DEV),
                      "exp_avg_sq": torch.zeros(n, device=DEV)} for i, n in enumerate(lengths)}


def twin_of(state, **kw):
    params = [torch.nn.Parameter(e["param"].double()) for e in state.values()]
    ref = torch.optim.AdamW(params, betas=(0.9, 0.999), eps=1e-8, **kw)
    for p, e in zip(params, state.values()):
        ref.state[p] = {"step": torch.tensor(float(e.get("step", 0))), "exp_avg": e["exp_avg"].double(),
                        "exp_avg_sq": e["exp_avg_sq"].double()}
    return params, ref


def run(state, opt, params, ref, present, g, lr):
    """K steps of both; ``present[k]`` names the parameters that have a gradient at step k."""
    for names in present:
        grads = {n: torch.randn(state[n]["param"].shape, generator=g, device=DEV) for n in names}
        for p, n in zip(params, state):
            p.grad = grads[n].double() if n in grads else None
        opt.step(grads)
        ref.step()
    K = len(present)
    for p, e in zip(params, state.values()):
        off = (e["param"].double() - p.detach()).abs()
        assert bool((off <= K * 16 * u * (p.detach().abs() + K * lr * 4)).all()), float(off.max())
    for p, e in zip(params, opt.state().values()):
        assert float(e["step"]) == float(ref.state[p]["step"])


@pytest.mark.parametrize("lengths", [[1000, 33, 5], [40, 2049, 1]])
def test_missing_gradients(lengths):
    """p1's first gradient comes at the fifth step, p2 has one now and then."""
    g = gen(1)
    state = fresh(g, lengths)
    params, ref = twin_of(state, lr=1e-2, weight_decay=0.05)
    opt = ShardAdamW(state, lr=1e-2, weight_decay=0.05)
    present = [["p0"], ["p0", "p2"], ["p0"], [], ["p0", "p1"], ["p0", "p1", "p2"], ["p0", "p1"], ["p1"],
               ["p0", "p1", "p2"], ["p0", "p1"]]
    run(state, opt, params, ref, present, g, 1e-2)
    assert opt.steps == 8 and [float(e["step"]) for e in opt.state().values()] == [8, 6, 3]


def test_a_state_whose_steps_differ_goes_on():
    g = gen(2)
    state = fresh(g, [300, 200, 100])
    for e, n in zip(state.values(), (3, 1000, 0)):
        e["step"] = torch.tensor(float(n))
        if n:
            e["exp_avg"].normal_(generator=g).mul_(0.1)
            e["exp_avg_sq"].uniform_(0.5, 1.5, generator=g)
    params, ref = twin_of(state, lr=1e-3, weight_decay=0.01)
    opt = ShardAdamW(state, lr=1e-3, weight_decay=0.01)
    assert opt.steps == 1000
    run(state, opt, params, ref, [list(state)] * 10, g, 1e-3)
    assert [float(e["step"]) for e in opt.state().values()] == [13, 1010, 10]
    again = ShardAdamW(opt.state())
    assert again.steps == 1010


def test_clipping_with_steps_that_differ():
    """The norm is that of all gradients, whatever their parameters' steps."""
    g = gen(3)
    state = fresh(g, [300, 200])
    alone = {n: {f: t.clone() for f, t in e.items()} for n, e in state.items()}
    state["p1"]["step"], alone["p1"]["step"] = torch.tensor(9.0), torch.tensor(9.0)
    grads = [torch.randn(n, generator=g, device=DEV) for n in (300, 200)]
    state["p0"]["step"] = alone["p0"]["step"] = torch.tensor(0.0)
    norm = ShardAdamW(state).step(grads, max_norm=0.5)
    q = sum(t.double().square().sum() for t in grads)
    for n, t in zip(alone, grads):
        got = ShardAdamW({n: alone[n]}).step([t], max_norm=0.5, square_sum=q)
        assert abs(float(got) - float(norm)) <= 2 * u * float(norm)
        for f in ("param", "exp_avg", "exp_avg_sq"):
            assert bool(((state[n][f] - alone[n][f]).abs() <= 8 * u * alone[n][f].abs()).all())


def test_step_fields():
    """A step field that entries share is parted where their counts differ;
    entries without one start where the others are, if these agree."""
    g = gen(4)
    state = fresh(g, [8, 8, 8])
    shared = torch.tensor(2.0)
    state["p0"]["step"] = state["p1"]["step"] = shared
    opt = ShardAdamW(state)
    opt.step({"p0": torch.ones(8, device=DEV)})
    opt.step({"p0": torch.ones(8, device=DEV), "p2": torch.ones(8, device=DEV)})
    assert [float(e["step"]) for e in opt.state().values()] == [4, 2, 3]
    opt.step({"p1": torch.ones(8, device=DEV)})
    assert [float(e["step"]) for e in opt.state().values()] == [4, 3, 3]
    opt.steps = 11
    assert opt.steps == 11 and [float(e["step"]) for e in opt.state().values()] == [11, 11, 11]


def test_names_of_one_tensor_count_together():
    g = gen(5)
    state = fresh(g, [8])
    state["head"] = dict(state["p0"])
    opt = ShardAdamW(state)
    opt.step({"p0": torch.ones(8, device=DEV)})
    opt.step({"head": torch.ones(8, device=DEV)})
    assert [float(e["step"]) for e in opt.state().values()] == [2, 2]
    with pytest.raises(PlanError, match="overlaps"):
        opt.step({n: torch.ones(8, device=DEV) for n in state})
    assert opt.steps == 2
    state["head"]["step"] = torch.tensor(5.0)
    with pytest.raises(PlanError, match="p0 and head are one tensor"):
        ShardAdamW(state)


def test_a_refused_step_does_not_count():
    state = fresh(gen(6), [8, 8])
    opt = ShardAdamW(state)
    with pytest.raises(PlanError):
        opt.step([torch.ones(8, device=DEV), torch.ones(7, device=DEV)])
    opt.step([torch.ones(8, device=DEV), None])
    assert [float(e["step"]) for e in opt.state().values()] == [1, 0]


def test_nothing_to_step():
    opt = ShardAdamW({})
    assert opt.step([]) is None and opt.steps == 0 and opt.state() == {}
    assert float(opt.step({}, max_norm=1.0)) == 0.0
    opt = ShardAdamW(fresh(gen(7), [8]))
    assert float(opt.step([None], max_norm=1.0)) == 0.0 and opt.steps == 0
