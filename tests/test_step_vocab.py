"""The vocabulary shard's operators without a GPU: what the C ABI refuses
before it launches anything, its workspaces, and what the torch entry points
refuse."""
import ctypes

import pytest
import torch

from suika_amd import PlanError, token_logprobs, vocab_embedding, vocab_embedding_grad
from suika_amd import _lib

vp, u64 = ctypes.c_void_p, ctypes.c_uint64
F32, BF16, F16, I32, I64 = (_lib.SR_DT_F32, _lib.SR_DT_BF16, _lib.SR_DT_F16, _lib.SR_DT_I32, _lib.SR_DT_I64)
BASE = 0x10000000     # an address that nothing reads: every call here is refused


class EmbeddingShape(ctypes.Structure):
    _fields_ = [("tokens", vp), ("token_dtype", ctypes.c_int32), ("dtype", ctypes.c_int32), ("n_tokens", u64),
                ("rows", u64), ("cols", u64), ("vocab_start", ctypes.c_int64), ("scale", ctypes.c_float),
                ("reserved", ctypes.c_int32)]


def embedding_shape(**kw):
    f = dict(tokens=BASE, token_dtype=I64, dtype=F32, n_tokens=4, rows=8, cols=16, vocab_start=0, scale=1.0,
             reserved=0)
    f.update(kw)
    return EmbeddingShape(**f)


def embedding(weight=BASE + 4096, stride=16, out=BASE + 65536, **kw):
    s = embedding_shape(**kw)
    return _lib.lib().sr_embedding(ctypes.byref(s), vp(weight), u64(stride), vp(out), None)


def embedding_grad(grad_out=BASE + 4096, stride=16, grad=BASE + 65536, grad_dtype=F32, work=BASE + (1 << 20),
                   work_bytes=1 << 20, **kw):
    s = embedding_shape(**kw)
    return _lib.lib().sr_embedding_grad(ctypes.byref(s), vp(grad_out), u64(stride), vp(grad), grad_dtype, 0, vp(work),
                                        u64(work_bytes), None)


@pytest.mark.parametrize("shape,code", [
    (dict(token_dtype=F32), _lib.SR_EDTYPE),
    (dict(dtype=_lib.SR_DT_F64), _lib.SR_EDTYPE),
    (dict(reserved=1), _lib.SR_EINVAL),
    (dict(tokens=None), _lib.SR_EINVAL),
    (dict(tokens=BASE + 4), _lib.SR_EALIGN),
    (dict(n_tokens=(1 << 23) + 1), _lib.SR_EBOUNDS),
    (dict(rows=(1 << 23) + 1), _lib.SR_EBOUNDS),
    (dict(cols=(1 << 23) + 1), _lib.SR_EBOUNDS),
])
def test_embedding_shapes_refused(shape, code):
    assert embedding(**shape) == code and _lib.last_error()
    assert embedding_grad(**shape) == code
    need = u64()
    assert _lib.lib().sr_embedding_grad_workspace(ctypes.byref(embedding_shape(**shape)), ctypes.byref(need)) == code


@pytest.mark.parametrize("kw,code", [
    (dict(weight=None), _lib.SR_EINVAL),
    (dict(out=None), _lib.SR_EINVAL),
    (dict(stride=15), _lib.SR_EINVAL),
    (dict(weight=BASE + 4098), _lib.SR_EALIGN),
    (dict(out=BASE + 65537), _lib.SR_EALIGN),
    (dict(out=BASE + 4096 + 8 * 64 - 4), _lib.SR_EOVERLAP),
    (dict(out=BASE + 16), _lib.SR_EOVERLAP),
])
def test_embedding_refused(kw, code):
    assert embedding(**kw) == code and "sr_embedding" in _lib.last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(grad_out=None), _lib.SR_EINVAL),
    (dict(grad=None), _lib.SR_EINVAL),
    (dict(grad_dtype=I32), _lib.SR_EDTYPE),
    (dict(stride=15), _lib.SR_EINVAL),
    (dict(grad=BASE + 65538), _lib.SR_EALIGN),
    (dict(work=None), _lib.SR_EINVAL),
    (dict(work_bytes=16), _lib.SR_EINVAL),
    (dict(work=BASE + (1 << 20) + 8), _lib.SR_EALIGN),
    (dict(grad=BASE + 4096 + 4 * 64 - 4), _lib.SR_EOVERLAP),
    (dict(grad=BASE), _lib.SR_EOVERLAP),
    (dict(work=BASE + 65536 + 16), _lib.SR_EOVERLAP),
    (dict(work=BASE + 4096 + 16), _lib.SR_EOVERLAP),
    (dict(work=BASE + 16), _lib.SR_EOVERLAP),
])
def test_embedding_grad_refused(kw, code):
    assert embedding_grad(**kw) == code and "sr_embedding_grad" in _lib.last_error()


def test_embedding_of_nothing():
    assert embedding(n_tokens=0, tokens=None) == 0
    assert embedding(cols=0, stride=0) == 0
    assert embedding_grad(rows=0) == 0
    assert embedding_grad(cols=0, stride=0) == 0


def test_torch_entry_points_refuse():
    tokens, weight = torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8)
    with pytest.raises(PlanError, match="GPU"):
        vocab_embedding(tokens, weight)
    with pytest.raises(PlanError, match="GPU"):
        vocab_embedding_grad(tokens, torch.zeros(3, 8), 4)
    with pytest.raises(PlanError, match="rows x columns"):
        vocab_embedding(tokens, weight[0])
    with pytest.raises(PlanError, match="tokens' shape"):
        vocab_embedding_grad(tokens, torch.zeros(2, 8), 4)


class LogprobShape(ctypes.Structure):
    _fields_ = [("logits", vp), ("targets", vp), ("target_dtype", ctypes.c_int32), ("dtype", ctypes.c_int32),
                ("rows", u64), ("columns", u64), ("vocab", u64), ("stride", u64)]


def logprob_shape(**kw):
    f = dict(logits=BASE, targets=BASE + (1 << 20), target_dtype=I64, dtype=F32, rows=4, columns=16, vocab=15,
             stride=16)
    f.update(kw)
    return LogprobShape(**f)


OUT = BASE + (1 << 21)


def logprob(top=2, out=(OUT, OUT + 64, OUT + 128, OUT + 192, OUT + 256), work=OUT + 4096, work_bytes=1 << 20, **kw):
    s = logprob_shape(**kw)
    return _lib.lib().sr_logprob(ctypes.byref(s), top, *[vp(p) for p in out], vp(work), u64(work_bytes), None)


def logprob_grad(lse=OUT, entropy=OUT + 64, gl=OUT + 128, gh=OUT + 192, grad=OUT + 4096, stride=16, **kw):
    s = logprob_shape(**kw)
    return _lib.lib().sr_logprob_grad(ctypes.byref(s), vp(lse), vp(entropy), vp(gl), vp(gh), vp(grad), u64(stride),
                                      None)


@pytest.mark.parametrize("shape,code", [
    (dict(target_dtype=F32), _lib.SR_EDTYPE),
    (dict(dtype=I64), _lib.SR_EDTYPE),
    (dict(rows=(1 << 23) + 1), _lib.SR_EBOUNDS),
    (dict(columns=(1 << 23) + 1, stride=1 << 24), _lib.SR_EBOUNDS),
    (dict(vocab=0), _lib.SR_EINVAL),
    (dict(vocab=17), _lib.SR_EINVAL),
    (dict(stride=15), _lib.SR_EINVAL),
    (dict(logits=None), _lib.SR_EINVAL),
    (dict(targets=None), _lib.SR_EINVAL),
    (dict(logits=BASE + 2), _lib.SR_EALIGN),
    (dict(targets=BASE + 4), _lib.SR_EALIGN),
])
def test_logprob_shapes_refused(shape, code):
    assert logprob(**shape) == code and _lib.last_error()
    assert logprob_grad(**shape) == code
    need = u64()
    assert _lib.lib().sr_logprob_workspace(ctypes.byref(logprob_shape(**shape)), 2, ctypes.byref(need)) == code


@pytest.mark.parametrize("kw,code", [
    (dict(top=-1), _lib.SR_EINVAL),
    (dict(top=65, columns=100, vocab=100, stride=100), _lib.SR_EINVAL),
    (dict(top=16), _lib.SR_EINVAL),                                   # more than the vocabulary
    (dict(out=(None, OUT, OUT, OUT, OUT)), _lib.SR_EINVAL),
    (dict(out=(OUT, OUT, OUT, None, OUT)), _lib.SR_EINVAL),
    (dict(out=(OUT, OUT + 2, OUT, OUT, OUT)), _lib.SR_EALIGN),
    (dict(out=(OUT, OUT, OUT, OUT, OUT + 4)), _lib.SR_EALIGN),
    (dict(work=OUT + 8), _lib.SR_EALIGN),
    (dict(out=(OUT, OUT + 12, OUT + 128, OUT + 192, OUT + 256)), _lib.SR_EOVERLAP),      # two outputs
    (dict(out=(OUT, OUT + 64, OUT + 128, OUT + 192, OUT + 208)), _lib.SR_EOVERLAP),
    (dict(out=(BASE + 4, OUT + 64, OUT + 128, OUT + 192, OUT + 256)), _lib.SR_EOVERLAP), # the logits
    (dict(out=(OUT, OUT + 64, OUT + 128, OUT + 192, BASE + (1 << 20) + 8)), _lib.SR_EOVERLAP),
])
def test_logprob_refused(kw, code):
    assert logprob(**kw) == code and "sr_logprob" in _lib.last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(lse=None), _lib.SR_EINVAL),
    (dict(entropy=None), _lib.SR_EINVAL),
    (dict(grad=None), _lib.SR_EINVAL),
    (dict(stride=15), _lib.SR_EINVAL),
    (dict(grad=OUT + 4098), _lib.SR_EALIGN),
    (dict(gl=OUT + 130), _lib.SR_EALIGN),
    (dict(grad=BASE + 4), _lib.SR_EOVERLAP),
    (dict(grad=BASE, stride=17), _lib.SR_EOVERLAP),
    (dict(grad=OUT + 8), _lib.SR_EOVERLAP),
    (dict(grad=BASE + (1 << 20)), _lib.SR_EOVERLAP),
])
def test_logprob_grad_refused(kw, code):
    assert logprob_grad(**kw) == code and "sr_logprob_grad" in _lib.last_error()


def test_logprob_of_nothing():
    assert logprob(rows=0, logits=None, targets=None) == 0
    assert logprob_grad(rows=0, logits=None, targets=None) == 0


def test_token_logprobs_refuses():
    with pytest.raises(PlanError, match="GPU"):
        token_logprobs(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(PlanError, match="targets' shape"):
        token_logprobs(torch.zeros(3, 5), torch.zeros(4, dtype=torch.int64))
