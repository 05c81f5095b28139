"""The sums, norms and workspaces of the optimizer operators overlap none of the
arrays that a call reads or writes: a workgroup would read what another has
written.  Refused before anything is launched."""
import ctypes

import pytest

from suika_amd import _lib

vp, u64 = ctypes.c_void_p, ctypes.c_uint64
F32 = _lib.SR_DT_F32
BASE = 0x10000000     # an address that nothing reads: every call here is refused
ELSEWHERE = BASE + (1 << 24)


class Array(ctypes.Structure):
    _fields_ = [("data", vp), ("n", u64), ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class Norm(ctypes.Structure):
    _fields_ = [("square_sum", vp), ("sum", vp), ("workspace", vp), ("workspace_bytes", u64), ("norm", vp)]


class AdamTensor(ctypes.Structure):
    _fields_ = [(f, vp) for f in ("weight", "exp_avg", "exp_avg_sq", "param", "grad")] + [
        ("n", u64)] + [(f, ctypes.c_int32) for f in ("weight_dtype", "moment_dtype", "grad_dtype", "reserved")]


class AdamOptions(ctypes.Structure):
    _fields_ = [(f, ctypes.c_double) for f in ("lr", "beta1", "beta2", "eps", "weight_decay")] + [
        ("step", ctypes.c_int64), ("max_norm", ctypes.c_double)]


N = 100_000           # elements of an array: its sum has parts
ARRAYS = (Array * 2)(Array(BASE, N, F32, 0), Array(BASE + (1 << 20), N, F32, 0))
INSIDE = BASE + (1 << 20) + 4 * N - 16      # the last elements of the second


def norm(square_sum=None, sum=ELSEWHERE, workspace=ELSEWHERE + 64, norm=ELSEWHERE + 8):
    return Norm(square_sum, sum, workspace, 1 << 16, norm)


@pytest.mark.parametrize("kw", [dict(sum=INSIDE), dict(norm=INSIDE), dict(workspace=INSIDE),
                                dict(norm=ELSEWHERE + 4), dict(workspace=ELSEWHERE),
                                dict(norm=ELSEWHERE + 72)])
def test_sums(kw):
    L, n = _lib.lib(), norm(**kw)
    assert L.sr_square_sum(ARRAYS, 2, 0, vp(n.workspace), u64(1 << 16), vp(n.sum), vp(n.norm), None) == _lib.SR_EOVERLAP
    assert "sr_square_sum" in _lib.last_error()
    assert L.sr_clip_norm(ARRAYS, None, 2, ctypes.c_float(1.0), ctypes.byref(n), None) == _lib.SR_EOVERLAP
    t = adam_tensor(grad=BASE + (1 << 20))
    o = AdamOptions(1e-3, 0.9, 0.99, 1e-8, 0.1, 1, 1.0)
    assert L.sr_adamw_norm((AdamTensor * 1)(t), None, 1, ctypes.byref(o), ctypes.byref(n), None) == _lib.SR_EOVERLAP


def adam_tensor(**kw):
    f = dict(weight=BASE + (4 << 20), exp_avg=BASE + (5 << 20), exp_avg_sq=BASE + (6 << 20), param=None,
             grad=BASE + (7 << 20), n=N, weight_dtype=F32, moment_dtype=F32, grad_dtype=F32, reserved=0)
    f.update(kw)
    return AdamTensor(**f)


@pytest.mark.parametrize("given", [BASE, INSIDE, BASE + 8])
def test_a_given_sum_is_not_clipped(given):
    L = _lib.lib()
    assert L.sr_clip(ARRAYS, None, 2, vp(given), ctypes.c_float(1.0), None, None) == _lib.SR_EOVERLAP
    n = norm(square_sum=given)
    assert L.sr_clip_norm(ARRAYS, None, 2, ctypes.c_float(1.0), ctypes.byref(n), None) == _lib.SR_EOVERLAP


def test_a_norm_in_an_array_or_in_its_sum():
    L = _lib.lib()
    for place in (INSIDE, ELSEWHERE + 4):
        assert L.sr_clip(ARRAYS, None, 2, vp(ELSEWHERE), ctypes.c_float(1.0), vp(place), None) == _lib.SR_EOVERLAP


@pytest.mark.parametrize("field", ["weight", "exp_avg", "exp_avg_sq"])
def test_a_given_sum_is_not_updated(field):
    L, t = _lib.lib(), adam_tensor()
    o = AdamOptions(1e-3, 0.9, 0.99, 1e-8, 0.1, 1, 1.0)
    place = getattr(t, field) + 4 * N - 8
    assert L.sr_adamw((AdamTensor * 1)(t), 1, ctypes.byref(o), vp(place), None) == _lib.SR_EOVERLAP
    n = norm(square_sum=place)
    assert L.sr_adamw_norm((AdamTensor * 1)(t), None, 1, ctypes.byref(o), ctypes.byref(n), None) == _lib.SR_EOVERLAP
