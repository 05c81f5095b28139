"""ShardAdamW on fields whose memory, shape or type was replaced after the
optimizer was made: what no longer fits its weight is refused on the host,
what fits is updated where it lies now."""
import pytest
import torch

from suika_amd import PlanError, ShardAdamW

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def state_of(n=64):
    w = torch.linspace(-1, 1, n, device=DEV)
    return {"w": {"param": w.to(BF16), "master": w, "exp_avg": torch.ones(n, device=DEV),
                  "exp_avg_sq": torch.ones(n, device=DEV), "step": torch.tensor(3.0)}}


SHAPES, KINDS = ["short", "long", "shape", "empty", "strided"], ["cpu", "type"]
MATCH = {"strided": "not contiguous", "cpu": "is on cpu", "type": "w: "}


# set_ keeps a tensor's device and type
@pytest.mark.parametrize("how,what", [("data", x) for x in SHAPES + KINDS] + [("set_", x) for x in SHAPES])
@pytest.mark.parametrize("field", ["param", "master", "exp_avg", "exp_avg_sq"])
def test_replaced_fields_are_refused(field, how, what):
    state = state_of()
    opt = ShardAdamW(state)
    t = state["w"][field]
    other = BF16 if t.dtype == F32 else F32
    new = {"short": lambda: torch.zeros(8, dtype=t.dtype, device=DEV),
           "long": lambda: torch.zeros(65, dtype=t.dtype, device=DEV),
           "shape": lambda: torch.zeros(8, 8, dtype=t.dtype, device=DEV),
           "empty": lambda: torch.zeros(0, dtype=t.dtype, device=DEV),
           "strided": lambda: torch.zeros(128, dtype=t.dtype, device=DEV)[::2],
           "cpu": lambda: torch.zeros(64, dtype=t.dtype),
           "type": lambda: torch.zeros(64, dtype=other, device=DEV)}[what]()
    if how == "data":
        t.data = new
    else:
        t.set_(new)
    before = {f: x.clone() for f, x in state["w"].items()}
    # a gradient like the weight, as it is now
    grad = torch.ones(state["w"]["master"].shape, device=DEV)
    with pytest.raises(PlanError, match=MATCH.get(what, "fields of different shapes")):
        opt.step([grad], max_norm=1.0)
    assert opt.steps == 3 and all(torch.equal(x, before[f]) for f, x in state["w"].items())


def test_replaced_memory_of_the_same_kind_is_used():
    state, twin = state_of(), state_of()
    opt, other = ShardAdamW(state), ShardAdamW(twin)
    old = {f: t.data for f, t in state["w"].items() if f != "step"}
    kept = {f: t.clone() for f, t in old.items()}
    for f, t in old.items():
        state["w"][f].data = t.clone()
    grad = torch.ones(64, device=DEV)
    opt.step([grad])
    other.step([grad])
    for f in old:
        assert torch.equal(state["w"][f], twin["w"][f]) and torch.equal(old[f], kept[f])
