"""Refusals and workspaces of the gated feed-forward block, without a GPU."""
import ctypes

import pytest
import torch

from suika_amd import PlanError, _lib, gated_ffn, gated_ffn_grad

U64, I32, VP = ctypes.c_uint64, ctypes.c_int32, ctypes.c_void_p
NAMES = ("x", "gate", "up", "down")


class Shape(ctypes.Structure):
    _fields_ = [(n, VP) for n in NAMES] + [(n, U64) for n in ("tokens", "hidden", "ffn")] + \
        [(n + "_stride", U64) for n in NAMES] + [("dtype", I32), ("activation", I32)]


class Grads(ctypes.Structure):
    _fields_ = [(n, VP) for n in NAMES]


def shape(tokens=4, hidden=8, ffn=16, at=1 << 20, dtype=_lib.SR_DT_BF16, activation=0, **other):
    s = Shape(tokens=tokens, hidden=hidden, ffn=ffn, x_stride=hidden, gate_stride=hidden, up_stride=hidden,
              down_stride=ffn, dtype=dtype, activation=activation)
    for i, n in enumerate(NAMES):
        setattr(s, n, at * (i + 1))
    for n, v in other.items():
        setattr(s, n, v)
    return s


def workspace(s, keep=0):
    need = U64()
    return _lib.lib().sr_ffn_workspace(ctypes.byref(s), keep, ctypes.byref(need)), need.value


def call(s, out=100 << 20, gate_out=0, up_out=0, work=200 << 20, size=None):
    need = workspace(s, 1 if gate_out else 0)[1] if size is None else size
    return _lib.lib().sr_ffn(ctypes.byref(s), VP(out), VP(gate_out), VP(up_out), VP(work), U64(need), None)


def test_workspace():
    rc, need = workspace(shape())
    assert rc == 0 and need >= 4 * 16 * 2
    assert workspace(shape(tokens=0)) == (0, 0)
    # rows that tiles cannot be loaded from are copied
    rc, odd = workspace(shape(tokens=100, hidden=9, ffn=15))
    assert rc == 0 and odd >= 2 * 16 * (100 + 100 + 15 + 15 + 9)


@pytest.mark.parametrize("bad,code", [
    (dict(dtype=_lib.SR_DT_F64), _lib.SR_EDTYPE), (dict(activation=3), _lib.SR_EINVAL),
    (dict(tokens=(1 << 23) + 1), _lib.SR_EBOUNDS), (dict(hidden=(1 << 20) + 1), _lib.SR_EBOUNDS),
    (dict(ffn=(1 << 20) + 1), _lib.SR_EBOUNDS), (dict(x_stride=7), _lib.SR_EINVAL), (dict(up_stride=7), _lib.SR_EINVAL),
    (dict(down=0), _lib.SR_EINVAL), (dict(gate=1), _lib.SR_EALIGN)])
def test_bad_shapes(bad, code):
    s = shape(**bad)
    assert workspace(s)[0] == code and call(s, size=1 << 30) == code
    g, need = Grads(1 << 30, 2 << 30, 3 << 30, 4 << 30), U64()
    assert _lib.lib().sr_ffn_grad_workspace(ctypes.byref(s), VP(5 << 30), U64(s.hidden), ctypes.byref(g),
                                            ctypes.byref(need)) == code


def test_bad_outputs():
    s = shape()
    assert call(s, out=0) == _lib.SR_EINVAL
    assert call(s, out=(100 << 20) + 1) == _lib.SR_EALIGN
    assert call(s, gate_out=300 << 20) == _lib.SR_EINVAL
    assert call(s, size=1) == _lib.SR_EINVAL
    assert call(s, work=0) == _lib.SR_EINVAL
    assert call(s, work=(200 << 20) + 8) == _lib.SR_EALIGN
    assert call(s, out=1 << 20) == _lib.SR_EOVERLAP                       # x
    assert call(s, out=(200 << 20) + 16) == _lib.SR_EOVERLAP              # the workspace
    assert call(s, gate_out=300 << 20, up_out=(300 << 20) + 4) == _lib.SR_EOVERLAP


def test_bad_gradients():
    s = shape()
    g = Grads(1 << 30, 2 << 30, 3 << 30, 4 << 30)
    need = U64()
    L = _lib.lib()

    def grad(g, a=5 << 30, b=6 << 30, dy=7 << 30, stride=8, work=8 << 30, size=None):
        rc = L.sr_ffn_grad_workspace(ctypes.byref(s), VP(dy), U64(stride), ctypes.byref(g), ctypes.byref(need))
        if rc:
            return rc
        return L.sr_ffn_grad(ctypes.byref(s), VP(a), VP(b), VP(dy), U64(stride), ctypes.byref(g), VP(work),
                             U64(need.value if size is None else size), None)

    assert grad(g, stride=7) == _lib.SR_EINVAL
    assert grad(g, a=0) == _lib.SR_EINVAL
    assert grad(g, b=2) == _lib.SR_EALIGN
    assert grad(g, dy=0) == _lib.SR_EINVAL
    assert grad(g, size=16) == _lib.SR_EINVAL
    assert grad(g, a=1 << 30) == _lib.SR_EOVERLAP
    assert grad(Grads(1 << 30, 2 << 30, 2 << 30, 4 << 30)) == _lib.SR_EOVERLAP
    assert grad(Grads(1 << 30, 2 << 30, 1, 4 << 30)) == _lib.SR_EALIGN


def test_refused_tensors():
    x, g, d = torch.zeros(4, 8), torch.zeros(16, 8), torch.zeros(8, 16)
    with pytest.raises(PlanError, match="not on the GPU"):
        gated_ffn(x, g, g, d)
    with pytest.raises(PlanError, match="not on the GPU"):
        gated_ffn_grad(x, g, g, d, torch.zeros(4, 16), torch.zeros(4, 16), x)
    with pytest.raises(PlanError, match="rows of hidden"):
        gated_ffn(torch.zeros(()), g, g, d)
    with pytest.raises(PlanError, match="wants a gradient"):
        gated_ffn(x.requires_grad_(), g, g, d, keep=True)
