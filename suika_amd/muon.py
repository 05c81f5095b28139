"""The Muon update of a share's matrices.

* ``orthogonalize``   -- matrices made orthogonal by Newton-Schulz products;
* ``ShardMuon``       -- momentum, the orthogonal update, decay, in place;
* ``split_matrices``  -- which matrices of a rank are parts of larger ones.

The matrices of a model's blocks are most of a share's state; the rest (norms,
biases, and as a rule the embedding and the head) is ``ShardAdamW``'s.  In the
reference all of it is ``torch.optim.AdamW``'s (tasks/task.py:72-73).

Where tensor parallelism cuts a matrix, its orthogonal update depends on all of
it.  A polynomial of the matrix needs only the products of its rows (or columns)
with each other, ``X^T X`` or ``X X^T``, and those of the parts add up: with
``split`` and ``all_reduce`` every rank keeps its part and exchanges these sums,
so a step's result depends on the degree only by the order of 32-bit sums.  The
products are then those of the side that is whole, whichever is shorter, and every
rank forms ``B`` by itself: where the cut side is much the shorter one, a whole
matrix takes fewer operations.

The kernels run on the tensors' device, on its current stream, behind the C ABI
of include/suika_step.h.  Refused arguments raise ``PlanError``.
"""
from __future__ import annotations

import math
from numbers import Real
from typing import Callable, Dict, Iterable, List, Mapping, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from ._lib import PlanError
from .meta import ParamLayout
from .optim import Grads

Triple = Tuple[float, float, float]
COEFFICIENTS: Triple = (3.4445, -4.7750, 2.0315)


def _schedule(steps: int, coefficients: Union[Triple, Sequence[Triple]]) -> List[float]:
    """The coefficients of all steps, one after another."""
    try:
        len(coefficients)       # no iterator: ShardMuon goes through them at every step
        rows = list(coefficients)
        rows = [rows] * steps if rows and isinstance(rows[0], Real) else [list(r) for r in rows]
        if len(rows) == steps and all(len(r) == 3 for r in rows):
            return [float(x) for r in rows for x in r]
    except (TypeError, ValueError):
        pass
    raise PlanError(f"coefficients: three numbers, or three for each of the {steps} steps")


def _tensors(given: Iterable[Tensor], what: str) -> List[Tensor]:
    """What may be an iterator, which can be gone through once."""
    try:
        each = iter(given)
    except TypeError:
        raise PlanError(f"{what}: a sequence of tensors is wanted") from None
    return list(each)


def orthogonalize(matrices: Iterable[Tensor], *, steps: int = 5,
                  coefficients: Union[Triple, Sequence[Triple]] = COEFFICIENTS, eps: float = 1e-7,
                  out: Optional[Iterable[Tensor]] = None, split: Optional[Sequence[Optional[int]]] = None,
                  all_reduce: Optional[Callable[[Tensor], object]] = None) -> List[Tensor]:
    """Each matrix G of a list with its singular values moved towards 1.

    ``X = G / max(|G|, eps)`` with the norm of all elements, then ``steps`` times
    ``X = a X + (b A + c A A) X`` with ``A = X X^T`` and a step's ``a, b, c`` from
    ``coefficients`` (one triple, or one for each step).  Singular vectors stay,
    a singular value s becomes ``a s + b s^3 + c s^5``; coefficients with which
    values between 0 and 1 get beyond 1.9 are refused.

    The matrices are float32, bfloat16 or float16 with dense rows at any
    distance, of any shapes, on one device; results are of the same types, or go
    to ``out``, which may be the matrices themselves.  Products are formed of 22
    bits a value in sums of 32 bits, and the result is rounded once.  A matrix of
    zeros stays zeros, one with NaN or infinity becomes NaN, and the others of
    the list are not touched by it.  Where ``eps`` is far above a matrix's norm,
    what is below 2^-38 after the division by it is lost.

    Not differentiable: a matrix or an ``out`` that wants a gradient is refused,
    as is a forward-mode tangent of either.

    ``split`` gives for each matrix ``None``, or the dimension along which ranks
    hold parts of it: 0 where the rows are dealt out, 1 the columns.  All ranks
    call with the same list; ``all_reduce`` gets 1-dim float32 and float64
    tensors on the device and sums them over the ranks in place, in the current
    stream's order (``torch.distributed.all_reduce``, for example).
    """
    matrices, out = _tensors(matrices, "matrices"), None if out is None else _tensors(out, "out")
    if torch.is_grad_enabled():
        for what, given in (("matrices", matrices), ("out", out or [])):
            if any(isinstance(m, Tensor) and m.requires_grad for m in given):
                raise PlanError(f"{what}: one wants a gradient, which orthogonalize does not have")
    return _lib.host().orthogonalize(matrices, out, split, steps, _schedule(steps, coefficients), float(eps), all_reduce)


def split_matrices(layout: ParamLayout, rank: int) -> Dict[str, Tuple[int, int]]:
    """The matrices of ``rank`` that tensor parallelism cuts: by name the
    dimension, and its size in the whole matrix (``ShardMuon``'s ``splits``)."""
    out = {}
    for name, meta in layout.layout[rank].items():
        if meta.tp_deg() > 1 and len(meta.shape) == 2:
            dim = meta.slice_dim() % 2
            out[name] = (dim, int(meta.shape[dim]))
    return out


class ShardMuon:
    """Muon on the matrices of a share's state, in place.

    ``state`` is (a part of) the dict that ``execute_param_transfer`` returns,
    with a two-dimensional ``param`` and an ``exp_avg`` for every name.  An entry
    with a float32 ``master`` is updated there and its bfloat16 ``param`` is
    rounded from it, to nearest even; without a ``master`` the ``param``, float32
    or bfloat16, is the weight itself.  ``exp_avg`` is float32 or bfloat16.  Other
    fields are left alone.  The optimizer keeps the tensors (an entry replaced in
    the dict later is not seen).

    An update by g: ``exp_avg = momentum exp_avg + (1 - momentum) g``, stored;
    ``G = momentum exp_avg + (1 - momentum) g``, or ``exp_avg`` without
    ``nesterov``; ``w = w (1 - lr weight_decay) - lr r X`` with X of G as
    ``orthogonalize`` forms it.  ``adjust_lr`` says what r is: ``"original"``
    ``sqrt(max(1, rows / columns))``, ``"match_rms_adamw"`` ``0.2 sqrt(max(rows,
    columns))``, ``"none"`` 1.  These are ``torch.optim.Muon``'s, with all in 32
    bits and the products as in ``orthogonalize``.

    ``splits`` names the matrices that are parts of larger ones, cut along a
    dimension (``split_matrices``); ``all_reduce`` is as for ``orthogonalize``,
    and every rank steps the same names, in the same order and with gradients for
    the same ones.  Rows and columns are then those of the whole matrix.
    """

    def __init__(self, state: Dict[str, Dict[str, Tensor]], *, lr: float = 1e-3, momentum: float = 0.95,
                 nesterov: bool = True, weight_decay: float = 0.1, ns_steps: int = 5,
                 ns_coefficients: Union[Triple, Sequence[Triple]] = COEFFICIENTS, eps: float = 1e-7,
                 adjust_lr: str = "original", splits: Optional[Mapping[str, Tuple[int, int]]] = None,
                 all_reduce: Optional[Callable[[Tensor], object]] = None):
        self.lr, self.momentum, self.nesterov, self.weight_decay = lr, momentum, nesterov, weight_decay
        self.ns_steps, self.ns_coefficients, self.eps, self.all_reduce = ns_steps, ns_coefficients, eps, all_reduce
        self.names = list(state)
        self._state = state
        splits = dict(splits or {})
        unknown = splits.keys() - state.keys()
        if unknown:
            raise PlanError(f"splits of unknown parameters: {sorted(unknown)[:4]}")
        weight, param, dims, scale = [], [], [], []
        for name, entry in state.items():
            for f in ("param", "exp_avg"):
                if f not in entry:
                    raise PlanError(f"{name}: no {f} in the state")
            master = entry.get("master")
            weight.append(entry["param"] if master is None else master)
            param.append(None if master is None else entry["param"])
            if weight[-1].dim() != 2:
                raise PlanError(f"{name}: a matrix is wanted, not {tuple(weight[-1].shape)}")
            dim, whole = splits.get(name, (None, 0))
            if dim not in (None, 0, 1) or (dim is not None and whole < weight[-1].shape[dim]):
                raise PlanError(f"{name}: split {(dim, whole)} of {tuple(weight[-1].shape)}")
            dims.append(-1 if dim is None else dim)
            scale.append(_scale(name, adjust_lr, *(whole if d == dim else weight[-1].shape[d] for d in (0, 1))))
        self._native = _lib.host().MuonState(weight, [e["exp_avg"] for e in state.values()], param, self.names, dims, scale)

    def step(self, grads: Union[Grads, Mapping[str, Optional[Tensor]]], *, max_norm: Optional[float] = None,
             square_sum: Optional[Tensor] = None) -> Optional[Tensor]:
        """One update by ``grads``: contiguous float32 or bfloat16 tensors in the
        order of ``names``, or by name; a parameter whose gradient is ``None``
        or missing keeps its state.

        With ``max_norm`` the gradients count as clipped to it (``clip_grads``;
        they are not written) and their norm is returned, a 0-dim float32
        tensor; ``square_sum`` is as for ``clip_grads``, and wanted where a matrix
        of ``splits`` is stepped: its parts are clipped alike.  An ``all_reduce`` that
        raises ends the step: all momentum is updated then, and the weights of
        matrices outside ``splits``; of the others' some, each as a whole.
        """
        if not isinstance(grads, (list, tuple)) and isinstance(grads, Mapping):
            unknown = grads.keys() - self._state.keys()
            if unknown:
                raise PlanError(f"gradients of unknown parameters: {sorted(unknown)[:4]}")
            grads = [grads.get(n) for n in self.names]
        return self._native.step(grads, self.lr, self.momentum, self.nesterov, self.weight_decay, self.ns_steps,
                                 _schedule(self.ns_steps, self.ns_coefficients), self.eps, max_norm, square_sum,
                                 self.all_reduce)

    def state(self) -> Dict[str, Dict[str, Tensor]]:
        """The state: the source of the next ``execute_param_transfer``."""
        return self._state


def _scale(name: str, adjust_lr: str, rows: int, columns: int) -> float:
    if adjust_lr == "original":
        return math.sqrt(max(1.0, rows / max(columns, 1)))
    if adjust_lr == "match_rms_adamw":
        return 0.2 * math.sqrt(max(rows, columns))
    if adjust_lr == "none":
        return 1.0
    raise PlanError(f"adjust_lr: {adjust_lr}, not original, match_rms_adamw or none")
