"""Gradient norm, clipping and AdamW without a GPU: what the C ABI refuses
before it launches anything, what the torch entry points refuse, and which
rank counts which gradient."""
import ctypes

import pytest
import torch

from suika_amd import (ParamLayout, PlanError, ShardAdamW, TensorMeta, clip_grads, counted_names, grad_norm,
                       grad_square_sum)
from suika_amd import _lib

vp = ctypes.c_void_p


class Array(ctypes.Structure):
    _fields_ = [("data", vp), ("n", ctypes.c_uint64), ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class AdamTensor(ctypes.Structure):
    _fields_ = [(f, vp) for f in ("weight", "exp_avg", "exp_avg_sq", "param", "grad")] + [
        ("n", ctypes.c_uint64)] + [(f, ctypes.c_int32) for f in ("weight_dtype", "moment_dtype", "grad_dtype",
                                                                 "reserved")]


class AdamOptions(ctypes.Structure):
    _fields_ = [(f, ctypes.c_double) for f in ("lr", "beta1", "beta2", "eps", "weight_decay")] + [
        ("step", ctypes.c_int64), ("max_norm", ctypes.c_double)]


F32, BF16, F16 = _lib.SR_DT_F32, _lib.SR_DT_BF16, _lib.SR_DT_F16
BASE = 0x10000000     # an address that nothing reads: every call here is refused


def arrays(*specs):
    return (Array * max(1, len(specs)))(*[Array(*s) for s in specs])


@pytest.mark.parametrize("spec,code", [
    ((BASE, 4, _lib.SR_DT_I32, 0), _lib.SR_EDTYPE),
    ((BASE, 4, _lib.SR_DT_F64, 0), _lib.SR_EDTYPE),
    ((BASE, 4, F32, 1), _lib.SR_EINVAL),
    ((None, 4, F32, 0), _lib.SR_EINVAL),
    ((BASE + 2, 4, F32, 0), _lib.SR_EALIGN),
    ((BASE + 1, 4, BF16, 0), _lib.SR_EALIGN),
    ((BASE, (1 << 34) + 1, F32, 0), _lib.SR_EBOUNDS),
])
def test_arrays_refused(spec, code):
    L = _lib.lib()
    need = ctypes.c_uint64()
    assert L.sr_square_sum_workspace(arrays(spec), 1, ctypes.byref(need)) == code
    assert L.sr_clip(arrays(spec), None, 1, vp(BASE), ctypes.c_float(1.0), None, None) == code
    assert _lib.last_error()


def test_square_sum_workspace():
    L = _lib.lib()
    need = ctypes.c_uint64()
    assert L.sr_square_sum_workspace(arrays(), 0, ctypes.byref(need)) == 0 and need.value == 0
    assert L.sr_square_sum_workspace(arrays((BASE, 0, F32, 0), (None, 0, BF16, 0)), 2, ctypes.byref(need)) == 0
    assert need.value == 0
    assert L.sr_square_sum_workspace(arrays((BASE, 5, F32, 0)), 1, ctypes.byref(need)) == 0
    assert need.value >= 8
    assert L.sr_square_sum_workspace(arrays(), -1, ctypes.byref(need)) == _lib.SR_EINVAL
    assert L.sr_square_sum_workspace(None, 1, ctypes.byref(need)) == _lib.SR_EINVAL
    one = arrays((BASE, 5, F32, 0))
    assert L.sr_square_sum(one, 1, 0, vp(BASE), ctypes.c_uint64(0), vp(BASE), None, None) == _lib.SR_EINVAL
    assert L.sr_square_sum(one, 1, 0, None, ctypes.c_uint64(1 << 20), vp(BASE), None, None) == _lib.SR_EINVAL
    assert L.sr_square_sum(one, 1, 0, vp(BASE + 8), ctypes.c_uint64(1 << 20), vp(BASE), None, None) == _lib.SR_EALIGN
    assert L.sr_square_sum(one, 1, 0, vp(BASE), ctypes.c_uint64(1 << 20), None, None, None) == _lib.SR_EINVAL
    assert L.sr_square_sum(one, 1, 0, vp(BASE), ctypes.c_uint64(1 << 20), vp(BASE + 4), None, None) == _lib.SR_EALIGN
    assert L.sr_square_sum(one, 1, 0, vp(BASE), ctypes.c_uint64(1 << 20), vp(BASE), vp(BASE + 2), None) == _lib.SR_EALIGN


def test_clip_refusals():
    L = _lib.lib()
    one = arrays((BASE, 8, F32, 0))

    def clip(src, dst, n, q=vp(BASE), max_norm=1.0):
        return L.sr_clip(src, dst, n, q, ctypes.c_float(max_norm), None, None)
    assert clip(one, None, 1, q=None) == _lib.SR_EINVAL
    assert clip(one, None, 1, q=vp(BASE + 4)) == _lib.SR_EALIGN
    assert clip(one, None, 1, max_norm=-1.0) == _lib.SR_EINVAL
    assert clip(one, None, 1, max_norm=float("nan")) == _lib.SR_EINVAL
    assert clip(one, arrays((BASE + 64, 7, F32, 0)), 1) == _lib.SR_EINVAL           # other length
    assert clip(one, arrays((BASE + 16, 8, F32, 0)), 1) == _lib.SR_EOVERLAP         # shifted onto itself
    assert clip(one, arrays((BASE, 8, BF16, 0)), 1) == _lib.SR_EOVERLAP             # the same memory, other type
    assert clip(arrays((BASE, 8, F32, 0), (BASE, 8, F32, 0)), None, 2) == _lib.SR_EOVERLAP     # listed twice
    two = arrays((BASE, 8, F32, 0), (BASE + 4096, 8, F32, 0))
    assert clip(two, arrays((BASE + 8192, 8, F32, 0), (BASE + 8208, 8, F32, 0)), 2) == _lib.SR_EOVERLAP
    assert clip(two, arrays((BASE + 4096, 8, F32, 0), (BASE + 8192, 8, F32, 0)), 2) == _lib.SR_EOVERLAP


def adam(options=None, **field):
    L = _lib.lib()
    f = dict(weight=BASE, exp_avg=BASE + 4096, exp_avg_sq=BASE + 8192, param=None, grad=BASE + 12288, n=8,
             weight_dtype=F32, moment_dtype=F32, grad_dtype=F32, reserved=0)
    f.update(field)
    o = dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1, step=1, max_norm=1.0)
    o.update(options or {})
    return L.sr_adamw((AdamTensor * 1)(AdamTensor(**f)), 1, ctypes.byref(AdamOptions(**o)), vp(BASE), None)


@pytest.mark.parametrize("options", [
    dict(lr=-1.0), dict(lr=float("nan")), dict(lr=float("inf")), dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0),
    dict(eps=-1e-8), dict(eps=float("nan")), dict(weight_decay=-1.0), dict(step=0), dict(max_norm=-1.0),
    dict(max_norm=float("nan")),
])
def test_adamw_options_refused(options):
    assert adam(options) == _lib.SR_EINVAL
    assert "sr_adamw" in _lib.last_error()


@pytest.mark.parametrize("field,code", [
    (dict(reserved=1), _lib.SR_EINVAL),
    (dict(weight_dtype=F16), _lib.SR_EDTYPE),
    (dict(moment_dtype=F16), _lib.SR_EDTYPE),
    (dict(grad_dtype=F16), _lib.SR_EDTYPE),
    (dict(weight_dtype=BF16, param=BASE + 16384), _lib.SR_EDTYPE),
    (dict(n=(1 << 34) + 1), _lib.SR_EBOUNDS),
    (dict(grad=None), _lib.SR_EINVAL),
    (dict(exp_avg=None), _lib.SR_EINVAL),
    (dict(weight=BASE + 2), _lib.SR_EALIGN),
    (dict(param=BASE + 16385), _lib.SR_EALIGN),
    (dict(exp_avg=BASE + 16), _lib.SR_EOVERLAP),
    (dict(param=BASE + 28), _lib.SR_EOVERLAP),
    (dict(grad=BASE + 16), _lib.SR_EOVERLAP),
])
def test_adamw_fields_refused(field, code):
    assert adam(**field) == code
    assert "sr_adamw" in _lib.last_error()


def test_adamw_refuses_a_tensor_listed_twice():
    one = AdamTensor(BASE, BASE + 4096, BASE + 8192, None, BASE + 12288, 8, F32, F32, F32, 0)
    o = AdamOptions(1e-3, 0.9, 0.99, 1e-8, 0.1, 1, 1.0)
    L = _lib.lib()
    assert L.sr_adamw((AdamTensor * 2)(one, one), 2, ctypes.byref(o), None, None) == _lib.SR_EOVERLAP
    assert L.sr_adamw(None, 1, ctypes.byref(o), None, None) == _lib.SR_EINVAL
    assert L.sr_adamw((AdamTensor * 1)(one), 1, None, None, None) == _lib.SR_EINVAL


@pytest.mark.parametrize("call", [grad_norm, grad_square_sum, lambda g: clip_grads(g, 1.0)])
def test_torch_entry_points_refuse(call):
    with pytest.raises(PlanError, match="cpu"):
        call([torch.zeros(3)])
    with pytest.raises(PlanError, match="not a tensor"):
        call([1.0])
    with pytest.raises(PlanError, match="sequence"):
        call(5)


def test_state_is_checked():
    t = torch.zeros(4)
    with pytest.raises(PlanError, match="exp_avg_sq"):
        ShardAdamW({"w": {"param": t, "exp_avg": t}})
    with pytest.raises(PlanError, match="steps differ"):
        ShardAdamW({"w": {"param": t, "exp_avg": t, "exp_avg_sq": t, "step": torch.tensor(3.0)},
                    "b": {"param": t, "exp_avg": t, "exp_avg_sq": t, "step": torch.tensor(4.0)}})
    with pytest.raises(PlanError, match="cpu"):
        ShardAdamW({"w": {"param": t, "exp_avg": t.clone(), "exp_avg_sq": t.clone()}})


def test_counted_names_count_every_shard_once():
    f = torch.float32
    layout = {}
    for dp in range(2):
        for tp in range(2):
            layout[2 * dp + tp] = {
                "w": TensorMeta(name="w", dtype=f, shape=(4, 4), tp_meta=(0, tp, 2)),
                "norm": TensorMeta(name="norm", dtype=f, shape=(4,)),
                "whole": TensorMeta(name="whole", dtype=f, shape=(4,), tp_meta=(0, 0, 1)),
            }
    layout[4] = {"last": TensorMeta(name="last", dtype=f, shape=(4,))}
    pl = ParamLayout.from_metas(layout)
    assert [counted_names(pl, r) for r in range(5)] == [["w", "norm", "whole"], ["w"], [], [], ["last"]]
