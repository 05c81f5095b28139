"""Refusals, workspaces and layouts of the Muon operators, without a GPU."""
import ctypes
import math

import pytest
import torch

from suika_amd import (QKV_HEADS, VOCAB_PAD, ParamLayout, PlanError, ShardMuon, TensorMeta, _lib, orthogonalize,
                       split_matrices)
from suika_amd.muon import COEFFICIENTS

U64, I64, I32, VP, F64 = ctypes.c_uint64, ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p, ctypes.c_double
REDUCE = ctypes.CFUNCTYPE(ctypes.c_int, VP, VP, U64, I32, VP)
BASE = 1 << 32


class Matrix(ctypes.Structure):
    _fields_ = [("data", VP), ("rows", U64), ("cols", U64), ("stride", U64), ("dtype", I32), ("split", I32)]


class Steps(ctypes.Structure):
    _fields_ = [("steps", I32), ("reserved", I32), ("coefficients", ctypes.POINTER(F64)), ("eps", F64), ("reduce", REDUCE),
                ("context", VP)]


class Tensor_(ctypes.Structure):
    _fields_ = [("weight", VP), ("exp_avg", VP), ("param", VP), ("grad", VP), ("rows", U64), ("cols", U64), ("scale", F64),
                ("weight_dtype", I32), ("moment_dtype", I32), ("grad_dtype", I32), ("split", I32), ("reserved", I64)]


class Options(ctypes.Structure):
    _fields_ = [("lr", F64), ("weight_decay", F64), ("momentum", F64), ("nesterov", I32), ("reserved", I32),
                ("max_norm", F64), ("square_sum", VP)]


def steps(n=5, coefficients=None, eps=1e-7, reduce=None, reserved=0):
    c = [x for _ in range(n) for x in COEFFICIENTS] if coefficients is None else coefficients
    return Steps(n, reserved, (F64 * max(1, len(c)))(*c), eps, reduce or REDUCE(0), None)


def matrix(rows=72, cols=80, at=0, dtype=_lib.SR_DT_F32, split=-1, stride=None):
    return Matrix(BASE + at, rows, cols, cols if stride is None else stride, dtype, split)


def workspace(src, dst=None, ns=None):
    dst = [matrix(m.rows, m.cols, (1 << 30) + (i << 24), m.dtype) for i, m in enumerate(src)] if dst is None else dst
    need = U64()
    ns = ns or steps()
    rc = _lib.lib().sr_orthogonalize_workspace((Matrix * max(1, len(src)))(*src), (Matrix * max(1, len(dst)))(*dst),
                                               len(src), ctypes.byref(ns), ctypes.byref(need))
    return rc, need.value


def test_workspace():
    assert workspace([]) == (0, 0)
    assert workspace([matrix(0, 5), matrix(5, 0, 1 << 20)]) == (0, 0)
    # X twice and A and B, as pairs of 16 bits with rows of whole 32s
    rc, need = workspace([matrix(100, 200)])
    assert rc == 0 and 100 * 4 * (2 * 224 + 2 * 128) <= need <= 100 * 4 * (2 * 224 + 2 * 128) + 4096
    assert workspace([matrix(200, 100)]) == (rc, need)
    # small ones stay in shared memory
    assert workspace([matrix(16, 24), matrix(64, 64, 1 << 20), matrix(700, 16, 2 << 20)]) == (0, 0)
    assert workspace([matrix(64, 65)])[1] > 0 and workspace([matrix(3200, 8)])[1] > 0
    # matrices beyond 8 GiB go one group after another, in the same memory
    big = [matrix(8192, 8192, i << 30, _lib.SR_DT_BF16) for i in range(12)]
    one, all_ = workspace(big[:8])[1], workspace(big, [matrix(8192, 8192, (100 + i) << 30, _lib.SR_DT_BF16) for i in range(12)])[1]
    assert one <= all_ < 1.01 * one


@pytest.mark.parametrize("bad,code", [
    (dict(dtype=_lib.SR_DT_I32), _lib.SR_EDTYPE), (dict(stride=15), _lib.SR_EINVAL), (dict(split=2), _lib.SR_EINVAL),
    (dict(split=0), _lib.SR_EINVAL), (dict(at=2), _lib.SR_EALIGN), (dict(rows=(1 << 19) + 1, cols=1), _lib.SR_EBOUNDS),
    (dict(rows=1 << 18, cols=1 << 18), _lib.SR_EBOUNDS)])
def test_bad_matrices(bad, code):
    assert workspace([matrix(**bad)])[0] == code


def test_bad_destinations():
    assert workspace([matrix()], [matrix(80, 72, 1 << 20)])[0] == _lib.SR_EINVAL
    assert workspace([matrix()], [matrix(at=64)])[0] == _lib.SR_EOVERLAP
    assert workspace([matrix()], [matrix()])[0] == 0                       # in place
    assert workspace([matrix(), matrix()], [matrix(), matrix()])[0] == _lib.SR_EOVERLAP
    assert workspace([matrix(), matrix(at=1 << 20)], [matrix(at=1 << 20), matrix()])[0] == _lib.SR_EOVERLAP
    need = workspace([matrix()])[1]
    L, ns = _lib.lib(), steps()
    src, dst = (Matrix * 1)(matrix()), (Matrix * 1)(matrix(at=1 << 20))
    assert L.sr_orthogonalize(src, dst, 1, ctypes.byref(ns), VP(1 << 40), U64(need - 1), None) == _lib.SR_EINVAL
    assert L.sr_orthogonalize(src, dst, 1, ctypes.byref(ns), VP((1 << 40) + 8), U64(need), None) == _lib.SR_EALIGN
    assert L.sr_orthogonalize(src, dst, 1, ctypes.byref(ns), VP(BASE + 16), U64(need), None) == _lib.SR_EOVERLAP


@pytest.mark.parametrize("bad", [
    dict(n=0), dict(n=65), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf), dict(reserved=1),
    dict(n=1, coefficients=[math.nan, 0, 0]), dict(n=1, coefficients=[math.inf, 0, 0]),
    dict(n=1, coefficients=[2.0, 0.0, 0.0]),                  # 1 becomes 2
    dict(n=2, coefficients=[1.5, 0.0, 0.0] * 2),              # 2.25 after two steps
    dict(n=1, coefficients=[6.0, -5.0, 0.0]),                 # 2.5 on the way to 1
    dict(n=1, coefficients=[1.0, 40.0, -40.0])])
def test_bad_steps(bad):
    assert workspace([matrix()], ns=steps(**bad))[0] == _lib.SR_EINVAL


@pytest.mark.parametrize("good", [
    dict(n=64), dict(n=1, coefficients=[1.875, -1.25, 0.375]), dict(n=3, coefficients=[1.5, -0.5, 0.0] * 3),
    dict(n=1, coefficients=[0.0, 0.0, 0.0]), dict(n=1, coefficients=[-1.0, 0.0, 0.0]), dict(eps=0.0),
    dict(n=2, coefficients=[3.9, -7.1, 4.1, 2.9, -3.1, 1.1])])
def test_good_steps(good):
    assert workspace([matrix()], ns=steps(**good))[0] == 0


def muon(tensors, options=None, ns=None):
    o = options or Options(1e-3, 0.1, 0.95, 1, 0, 0.0, None)
    need = U64()
    ns = ns or steps()
    return _lib.lib().sr_muon_workspace((Tensor_ * max(1, len(tensors)))(*tensors), len(tensors), ctypes.byref(o),
                                        ctypes.byref(ns), ctypes.byref(need)), need.value


def tensor(i=0, rows=72, cols=80, **other):
    at = BASE + (i << 28)
    t = Tensor_(at, at + (1 << 24), at + (2 << 24), at + (3 << 24), rows, cols, 1.0, _lib.SR_DT_F32, _lib.SR_DT_F32,
                _lib.SR_DT_BF16, -1, 0)
    for k, v in other.items():
        setattr(t, k, v)
    return t


def test_muon_workspace():
    rc, need = muon([tensor()])
    assert rc == 0 and need == workspace([matrix()])[1]
    assert muon([]) == (0, 0) and muon([tensor(rows=0)]) == (0, 0)
    assert muon([tensor(param=None, weight_dtype=_lib.SR_DT_BF16)])[0] == 0


@pytest.mark.parametrize("bad,code", [
    (dict(weight=None), _lib.SR_EINVAL), (dict(grad=None), _lib.SR_EINVAL), (dict(exp_avg=None), _lib.SR_EINVAL),
    (dict(weight_dtype=_lib.SR_DT_BF16), _lib.SR_EDTYPE), (dict(moment_dtype=_lib.SR_DT_F16), _lib.SR_EDTYPE),
    (dict(grad_dtype=_lib.SR_DT_F16), _lib.SR_EDTYPE), (dict(scale=-1.0), _lib.SR_EINVAL),
    (dict(scale=math.inf), _lib.SR_EINVAL), (dict(reserved=1), _lib.SR_EINVAL), (dict(split=1), _lib.SR_EINVAL),
    (dict(grad=BASE), _lib.SR_EOVERLAP), (dict(param=BASE + 4), _lib.SR_EOVERLAP), (dict(exp_avg=BASE + 2), _lib.SR_EALIGN)])
def test_bad_muon_tensors(bad, code):
    assert muon([tensor(**bad)])[0] == code


def test_bad_muon_options():
    for o in [(-1.0, 0.1, 0.9), (math.inf, 0.1, 0.9), (1e-3, -0.1, 0.9), (1e-3, 0.1, 1.0), (1e-3, 0.1, -0.1), (1e-3, math.nan, 0.9)]:
        assert muon([tensor()], Options(*o, 1, 0, 0.0, None))[0] == _lib.SR_EINVAL
    assert muon([tensor()], Options(1e-3, 0.1, 0.9, 1, 1, 0.0, None))[0] == _lib.SR_EINVAL
    assert muon([tensor()], Options(1e-3, 0.1, 0.9, 1, 0, -1.0, 1 << 40))[0] == _lib.SR_EINVAL
    assert muon([tensor()], Options(1e-3, 0.1, 0.9, 1, 0, 1.0, (1 << 40) + 4))[0] == _lib.SR_EALIGN
    assert muon([tensor()], Options(1e-3, 0.1, 0.9, 1, 0, 1.0, BASE + 8))[0] == _lib.SR_EOVERLAP


def state(shape=(8, 16), **other):
    return {"w": {"param": torch.zeros(shape), "exp_avg": torch.zeros(shape), **other}}


def test_refused_python_arguments():
    with pytest.raises(PlanError, match="not on the GPU"):
        orthogonalize([torch.zeros(3, 3)])
    with pytest.raises(PlanError, match="three numbers"):
        orthogonalize([], steps=2, coefficients=[(1.0, 0.0, 0.0)])
    with pytest.raises(PlanError, match="split has"):
        orthogonalize([], split=[0])
    with pytest.raises(PlanError, match="no exp_avg"):
        ShardMuon({"w": {"param": torch.zeros(2, 2)}})
    with pytest.raises(PlanError, match="a matrix is wanted"):
        ShardMuon(state((8,)))
    with pytest.raises(PlanError, match="splits of unknown"):
        ShardMuon(state(), splits={"v": (0, 16)})
    with pytest.raises(PlanError, match="split"):
        ShardMuon(state(), splits={"w": (2, 16)})
    with pytest.raises(PlanError, match="split"):
        ShardMuon(state(), splits={"w": (1, 15)})
    with pytest.raises(PlanError, match="adjust_lr"):
        ShardMuon(state(), adjust_lr="adam")
    with pytest.raises(PlanError, match="not a dense tensor on the GPU"):
        ShardMuon(state())


def test_split_matrices():
    bf16 = torch.bfloat16
    metas = {r: {
        "wte.weight": TensorMeta(name="wte.weight", dtype=bf16, shape=(100, 16), tp_meta=(0, r, 2), kind=VOCAB_PAD, kind_args=(8,)),
        "qkv.weight": TensorMeta(name="qkv.weight", dtype=bf16, shape=(32, 16), tp_meta=(0, r, 2), kind=QKV_HEADS,
                                 kind_args=(4, 2, 4)),
        "down.weight": TensorMeta(name="down.weight", dtype=bf16, shape=(16, 64), tp_meta=(-1, r, 2)),
        "bias": TensorMeta(name="bias", dtype=bf16, shape=(32,), tp_meta=(0, r, 2)),
        "norm.weight": TensorMeta(name="norm.weight", dtype=bf16, shape=(16,)),
        "whole.weight": TensorMeta(name="whole.weight", dtype=bf16, shape=(16, 16)),
    } for r in range(2)}
    layout = ParamLayout.from_metas(metas)
    assert split_matrices(layout, 1) == {"wte.weight": (0, 100), "qkv.weight": (0, 32), "down.weight": (1, 64)}
    one = ParamLayout.from_metas({0: {"a": TensorMeta(name="a", dtype=bf16, shape=(4, 4))}})
    assert split_matrices(one, 0) == {}


def test_matrices_from_an_iterator():
    """What can be gone through once reaches the host whole, in either mode."""
    for mode in (torch.enable_grad, torch.no_grad):
        with mode():
            with pytest.raises(PlanError, match=r"matrices\[0\] is on cpu"):
                orthogonalize(iter([torch.zeros(3, 3)]))
            with pytest.raises(PlanError, match="a sequence of tensors"):
                orthogonalize(None)
            with pytest.raises(PlanError, match="not a tensor"):
                orthogonalize(x for x in (1, 2))
    with pytest.raises(PlanError, match="wants a gradient"):
        orthogonalize(iter([torch.zeros(3, 3), torch.zeros(3, 3, requires_grad=True)]))


def test_outputs_that_want_a_gradient():
    g, out = torch.zeros(3, 3), torch.zeros(3, 3, requires_grad=True)
    for given in ([out], (out,), iter([out]), [out * 2]):
        with pytest.raises(PlanError, match="out: one wants a gradient"):
            orthogonalize([g], out=given)
    with torch.no_grad(), pytest.raises(PlanError, match="not on the GPU"):
        orthogonalize([g], out=[out])
    with pytest.raises(PlanError, match="out: a sequence of tensors"):
        orthogonalize([g], out=1)


def test_coefficients_of_any_kind():
    import numpy as np
    from suika_amd.muon import _schedule
    triple = (1.5, -0.5, 0.0)
    for given in (triple, list(triple), np.array(triple), np.array(triple, dtype=np.float32), [triple] * 2,
                  np.array([triple] * 2, dtype=np.float32)):
        assert _schedule(2, given) == list(triple) * 2
    for bad in ([], (), None, 1.5, "abc", iter(triple), triple[:2], [triple], [triple, None], [triple, ("a", "b", "c")], [[]] * 2):
        with pytest.raises(PlanError, match="three numbers"):
            orthogonalize([], steps=2, coefficients=bad)


def test_workspace_of_split_matrices():
    """X twice, A and B as pairs of 16 bits, and A in floats; groups of 8 GiB are counted without X."""
    ns = steps(reduce=REDUCE(lambda *a: 0))
    rc, need = workspace([matrix(100, 200, split=0)], ns=ns)
    exact = 4 * (2 * 200 * 128 + 2 * 200 * 224 + 200 * 200)
    assert rc == 0 and exact <= need <= exact + 4096
    rc, other = workspace([matrix(100, 200, split=1)], ns=ns)
    assert rc == 0 and 4 * (2 * 100 * 224 + 2 * 100 * 128 + 100 * 100) <= other < need
    wide = [matrix(4096, 65536, i << 32, split=1) for i in range(40)]
    rc, need = workspace(wide, [matrix(4096, 65536, (100 + i) << 32) for i in range(40)], ns)
    assert rc == 0 and need > 40 * 4 * (2 * 4096 * 65536 + 3 * 4096 * 4096)
