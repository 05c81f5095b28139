"""A vocabulary shard starts at a token: negative starts, which would make rows
of negative tokens, are refused before anything is launched."""
import ctypes

import pytest

from suika_amd import _lib

vp, u64 = ctypes.c_void_p, ctypes.c_uint64
BASE = 0x10000000     # an address that nothing reads: every call here is refused or has no tokens


class EmbeddingShape(ctypes.Structure):
    _fields_ = [("tokens", vp), ("token_dtype", ctypes.c_int32), ("dtype", ctypes.c_int32), ("n_tokens", u64),
                ("rows", u64), ("cols", u64), ("vocab_start", ctypes.c_int64), ("scale", ctypes.c_float),
                ("reserved", ctypes.c_int32)]


def shape(start, n=4):
    return EmbeddingShape(BASE, _lib.SR_DT_I64, _lib.SR_DT_F32, n, 8, 16, start, 1.0, 0)


@pytest.mark.parametrize("start", [-1, -8, -2 ** 62, -2 ** 63])
def test_negative_starts(start):
    L, s, need = _lib.lib(), shape(start), u64()
    assert L.sr_embedding(ctypes.byref(s), vp(BASE + 4096), u64(16), vp(BASE + 65536), None) == _lib.SR_EINVAL
    assert "vocab_start" in _lib.last_error()
    assert L.sr_embedding_grad_workspace(ctypes.byref(s), ctypes.byref(need)) == _lib.SR_EINVAL
    assert L.sr_embedding_grad(ctypes.byref(s), vp(BASE + 4096), u64(16), vp(BASE + 65536), _lib.SR_DT_F32, 0,
                               vp(BASE + (1 << 20)), u64(1 << 20), None) == _lib.SR_EINVAL


@pytest.mark.parametrize("start", [0, 8, 2 ** 62])
def test_starts_that_are_taken(start):
    L, need = _lib.lib(), u64()
    assert L.sr_embedding_grad_workspace(ctypes.byref(shape(start)), ctypes.byref(need)) == 0 and need.value > 0
    nothing = shape(start, 0)
    assert L.sr_embedding(ctypes.byref(nothing), vp(BASE + 4096), u64(16), vp(BASE + 65536), None) == 0
