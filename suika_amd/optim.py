"""The optimizer's part of a training step on a share's state.

Between two plan changes a job trains on the state that
``execute_param_transfer`` returns: ``{name: {"param", "exp_avg",
"exp_avg_sq"[, "master"][, "step"]}}``.  These operators work on that state as
it is, whatever allocation its tensors lie in:

* ``grad_norm`` / ``grad_square_sum`` -- the gradients' global 2-norm, or the
  sum of squares that ranks with other shards add up first;
* ``clip_grads``  -- the gradients scaled down to a norm;
* ``ShardAdamW``  -- norm, clipping and the AdamW update of every field.

In the reference this is ``torch.optim.AdamW`` over the model's parameters
(tasks/task.py:72-73).  The kernels run on the tensors' device, on its current
stream, behind the C ABI of include/suika_step.h; nothing synchronises with
the host.  Refused arguments raise ``PlanError`` before anything runs.
"""
from __future__ import annotations

from typing import Dict, List, Mapping, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from ._lib import PlanError
from .meta import ParamLayout

Grads = Sequence[Optional[Tensor]]


def grad_square_sum(grads: Grads) -> Tensor:
    """The sum of the squares of all elements of ``grads``, a 0-dim float64
    tensor on their device.

    ``grads`` are contiguous float32, bfloat16 or float16 tensors of any
    shapes; ``None`` stands for a parameter without gradient.  Squares and
    sums are computed in 64 bits, in an order that does not change from run to
    run.  Of a sharded model, each rank sums the gradients it counts
    (``counted_names``) and the ranks add their sums up.
    """
    return _lib.host().grad_square_sum(grads)


def grad_norm(grads: Grads) -> Tensor:
    """The 2-norm of all elements of ``grads`` together: the root of
    ``grad_square_sum``, a 0-dim float32 tensor."""
    return _lib.host().grad_norm(grads)


def clip_grads(grads: Grads, max_norm: float, *, out: Optional[Grads] = None,
               square_sum: Optional[Tensor] = None) -> Tensor:
    """Scale ``grads`` by ``min(1, max_norm / (norm + 1e-6))`` and return the
    norm that they had, a 0-dim float32 tensor.

    In place, where a factor of 1 leaves the memory as it is; or into the
    tensors of ``out``, of the same shapes and of any of the three types
    (bfloat16 gradients of a model into the float32 ones of its optimizer).
    ``square_sum`` is the sum to clip by where other ranks have a part in it
    (a float64 tensor, ``grad_square_sum`` added up over the ranks); by
    default that of ``grads``.  A norm that is NaN makes every gradient NaN;
    an infinite one makes the finite gradients 0, as
    ``torch.nn.utils.clip_grad_norm_`` does.
    """
    return _lib.host().clip_grads(grads, float(max_norm), out, square_sum)


def counted_names(layout: ParamLayout, rank: int) -> List[str]:
    """The parameters whose gradients ``rank`` counts in a global norm.

    Every element of a parameter is counted once.  Of its holders, those of one
    tensor-parallel degree count, each shard on the lowest rank that has it: so
    a tensor-parallel shard counts on each rank of one group, a replicated
    parameter (norms, row-parallel biases, data-parallel copies) on one rank.
    Where replicas hold a parameter at different degrees, the degree is that of
    the lowest rank whose degree's shards are all there.
    """
    mine = layout.layout[rank]
    holders: Dict[str, List[Tuple[int, int, int]]] = {n: [] for n in mine}     # (degree, index, rank), by rank
    for r in sorted(layout.layout):
        for n, m in layout.layout[r].items():
            if n in mine:
                holders[n].append((m.tp_deg(), m.tp_index(), r))
    return [n for n in mine if _counts(holders[n], rank)]


def _counts(holders: List[Tuple[int, int, int]], rank: int) -> bool:
    first: Dict[int, Dict[int, int]] = {}      # degree -> index -> the lowest rank that holds it
    for deg, index, r in holders:
        first.setdefault(deg, {}).setdefault(index, r)
    whole = [shards for deg, shards in first.items() if len(shards) == deg]
    return rank in (whole or list(first.values()))[0].values()


class ShardAdamW:
    """AdamW on a share's state, in place.

    ``state`` is the dict that ``execute_param_transfer`` returns.  An entry
    with a float32 ``master`` is updated there and its bfloat16 ``param`` is
    rounded from it, to nearest even; without a ``master`` the ``param``,
    float32 or bfloat16, is the weight itself.  The moments are both float32
    or both bfloat16.  Everything is computed in 32 bits and rounded where it
    is stored.  The optimizer keeps the tensors (an entry replaced in the dict
    later is not seen).

    Every parameter counts its own updates, from its ``step`` field on (where
    it has none: from the others' if they agree, else from 0), and one that
    gets no gradient does not count, as in ``torch.optim.AdamW``.  Names of one
    tensor count together, so their ``step`` fields have to agree.

    A parameter's update t, with g clipped: ``exp_avg = beta1 exp_avg +
    (1 - beta1) g``; ``exp_avg_sq = beta2 exp_avg_sq + (1 - beta2) g^2``;
    ``w = w (1 - lr weight_decay) - lr / (1 - beta1^t) exp_avg /
    (sqrt(exp_avg_sq / (1 - beta2^t)) + eps)``.
    """

    def __init__(self, state: Dict[str, Dict[str, Tensor]], *, lr: float = 1e-3,
                 betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01):
        self.lr, self.betas, self.eps, self.weight_decay = lr, tuple(betas), eps, weight_decay
        self.names = list(state)
        self._state = state
        weight, param = [], []
        counts: Dict[int, Tuple[str, int]] = {}      # of a tensor: a name of it, and its updates
        for name, entry in state.items():
            for f in ("param", "exp_avg", "exp_avg_sq"):
                if f not in entry:
                    raise PlanError(f"{name}: no {f} in the state")
            master = entry.get("master")
            weight.append(entry["param"] if master is None else master)
            param.append(None if master is None else entry["param"])
            if "step" in entry:
                step = int(entry["step"])
                other, count = counts.setdefault(id(weight[-1]), (name, step))
                if count != step:
                    raise PlanError(f"{other} and {name} are one tensor, but their steps differ: {count} and {step}")
        known = {count for _, count in counts.values()}
        rest = ("", known.pop() if len(known) == 1 else 0)
        self._native = _lib.host().AdamWState(weight, [e["exp_avg"] for e in state.values()],
                                              [e["exp_avg_sq"] for e in state.values()], param, self.names,
                                              [counts.get(id(w), rest)[1] for w in weight])

    @property
    def steps(self) -> int:
        """The most updates that a parameter has had; setting it sets all."""
        return max(self._native.steps, default=0)

    @steps.setter
    def steps(self, count: int) -> None:
        self._native.steps = [count] * len(self.names)

    def step(self, grads: Union[Grads, Mapping[str, Optional[Tensor]]], *, max_norm: Optional[float] = None,
             square_sum: Optional[Tensor] = None) -> Optional[Tensor]:
        """One update by ``grads``: contiguous float32 or bfloat16 tensors in the
        order of ``names``, or by name; a parameter whose gradient is ``None``
        or missing keeps its state, its step included.

        With ``max_norm`` the gradients count as clipped to it
        (``clip_grads``; they are not written) and their norm is returned, a
        0-dim float32 tensor; ``square_sum`` is as for ``clip_grads``.  The
        number of the step is a host value, so the call refuses to be captured
        into a graph.
        """
        if not isinstance(grads, (list, tuple)) and isinstance(grads, Mapping):
            unknown = grads.keys() - self._state.keys()
            if unknown:
                raise PlanError(f"gradients of unknown parameters: {sorted(unknown)[:4]}")
            grads = [grads.get(n) for n in self.names]
        return self._native.step(grads, self.lr, self.betas[0], self.betas[1], self.eps, self.weight_decay, max_norm,
                                 square_sum)

    def state(self) -> Dict[str, Dict[str, Tensor]]:
        """The state with its ``step`` fields brought up to date, each to its
        parameter's count: the source of the next ``execute_param_transfer``."""
        written: Dict[int, int] = {}
        for name, count in zip(self.names, self._native.steps):
            entry = self._state[name]
            old = entry.get("step")
            if not isinstance(old, Tensor):
                entry["step"] = torch.tensor(float(count))
            elif written.setdefault(id(old), count) == count:
                old.fill_(count)
            else:       # the same tensor as another entry's, which has had other updates
                entry["step"] = torch.full_like(old, count)
        return self._state
