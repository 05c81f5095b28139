"""A call of the optimizer operators that is refused launches nothing: in a
capture the graph stays empty, also where the call would have formed the
gradients' norm first."""
import warnings

import pytest
import torch

from suika_amd import PlanError, ShardAdamW, clip_grads

pytestmark = pytest.mark.gpu
DEV = "cuda"


def graph_is_empty(call):
    """Captures ``call``; whether torch says that the graph is empty, and what was raised."""
    graph, error = torch.cuda.CUDAGraph(), None
    torch.set_warn_always(True)
    try:
        with warnings.catch_warnings(record=True) as seen:
            warnings.simplefilter("always")
            try:
                with torch.cuda.graph(graph):
                    call()
            except PlanError as e:
                error = e
    finally:
        torch.set_warn_always(False)
    torch.cuda.synchronize()
    return any("empty" in str(w.message) for w in seen), error


def state_of():
    return {"w": {f: torch.ones(70000, device=DEV) for f in ("param", "exp_avg", "exp_avg_sq")}}


def test_refused_calls_launch_nothing():
    grad, other = torch.ones(70000, device=DEV), torch.ones(8, device=DEV)
    empty, error = graph_is_empty(lambda: clip_grads([grad], 1.0))
    assert not empty and error is None
    opt = ShardAdamW(state_of())
    for call, match in [(lambda: opt.step([grad], max_norm=1.0), "captured"),
                        (lambda: opt.step([grad], max_norm=1.0, square_sum=other), "square_sum"),
                        (lambda: opt.step([opt._state["w"]["param"]], max_norm=1.0), "overlaps"),
                        (lambda: opt.step([grad], max_norm=-1.0), "max_norm"),
                        (lambda: clip_grads([grad, grad], 1.0), "overlaps"),
                        (lambda: clip_grads([grad], 1.0, out=[]), "0 tensors"),
                        (lambda: clip_grads([grad, other], -1.0), "max_norm")]:
        empty, error = graph_is_empty(call)
        assert empty and error is not None and match in str(error), match
    assert opt.steps == 0


def test_a_refused_capture_by_a_given_sum_launches_nothing():
    opt, grad = ShardAdamW(state_of()), torch.ones(70000, device=DEV)
    q = torch.ones((), dtype=torch.float64, device=DEV)
    empty, error = graph_is_empty(lambda: opt.step([grad], max_norm=1.0, square_sum=q))
    assert empty and "captured" in str(error)
