"""CPU: the operators on device tensors refuse bad arguments before they look for a device.

No pointer here is ever followed: every call is refused on the host.
"""
import ctypes as C

import pytest
import torch

from loki_b200 import _lib, ops

P = C.c_void_p(4096)   # aligned to everything
ODD = C.c_void_p(4097)
F32, F16, I8, BF16 = _lib.LK_F32, _lib.LK_F16, _lib.LK_I8, _lib.LK_BF16


def norm(**kw):
    a = dict(device=0, dtype=F32, rows=4, dim=8, x=P, ldx=8, r=None, ldr=0, g=None, gt=0, eps=1e-6, s=None, lds=0, c=P, ldc=8, sc=P, st=None)
    a.update(kw)
    return _lib.lib.lk_rms_norm_i8(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=I8), _lib.LK_EINVAL), (dict(dtype=9), _lib.LK_EINVAL), (dict(g=P, gt=I8), _lib.LK_EINVAL),
    (dict(rows=-1), _lib.LK_EINVAL), (dict(dim=0), _lib.LK_EINVAL), (dict(dim=32769, ldx=32769, ldc=32769), _lib.LK_ERANGE),
    (dict(rows=1 << 31), _lib.LK_ERANGE), (dict(eps=-1.0), _lib.LK_EINVAL), (dict(eps=float("nan")), _lib.LK_EINVAL),
    (dict(eps=float("inf")), _lib.LK_EINVAL), (dict(x=None), _lib.LK_EINVAL), (dict(c=None), _lib.LK_EINVAL), (dict(sc=None), _lib.LK_EINVAL),
    (dict(ldx=7), _lib.LK_EINVAL), (dict(ldc=7), _lib.LK_EINVAL), (dict(r=P, ldr=7), _lib.LK_EINVAL), (dict(s=P, lds=7), _lib.LK_EINVAL),
    (dict(x=ODD), _lib.LK_EINVAL), (dict(r=ODD, ldr=8), _lib.LK_EINVAL), (dict(s=ODD, lds=8), _lib.LK_EINVAL),
    (dict(g=ODD, gt=BF16), _lib.LK_EINVAL), (dict(sc=ODD), _lib.LK_EINVAL), (dict(device=-1), _lib.LK_ECUDA), (dict(device=4096), _lib.LK_ECUDA),
])
def test_rms_norm_refuses(kw, status):
    assert norm(**kw) == status
    assert b"lk_rms_norm_i8" in _lib.lib.lk_last_error()


def linear(**kw):
    a = dict(device=0, dtype=I8, m=4, n=4, k=16, a=P, lda=16, sa=None, w=P, ldw=16, sw=None, bias=None, act=0, r=None, ldr=0, ot=F32, out=P, ldo=4, st=None)
    a.update(kw)
    return _lib.lib.lk_linear(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=F32), _lib.LK_EINVAL), (dict(ot=I8), _lib.LK_EINVAL), (dict(act=5), _lib.LK_EINVAL), (dict(act=-1), _lib.LK_EINVAL),
    (dict(m=-1), _lib.LK_EINVAL), (dict(n=-1), _lib.LK_EINVAL), (dict(k=-1), _lib.LK_EINVAL),
    (dict(k=65537, lda=65537, ldw=65537), _lib.LK_ERANGE), (dict(m=1 << 31), _lib.LK_ERANGE), (dict(n=1 << 31, ldo=1 << 31), _lib.LK_ERANGE),
    (dict(a=None), _lib.LK_EINVAL), (dict(w=None), _lib.LK_EINVAL), (dict(out=None), _lib.LK_EINVAL),
    (dict(lda=15), _lib.LK_EINVAL), (dict(ldw=15), _lib.LK_EINVAL), (dict(ldo=3), _lib.LK_EINVAL), (dict(r=P, ldr=3), _lib.LK_EINVAL),
    (dict(dtype=F16, a=ODD), _lib.LK_EINVAL), (dict(dtype=BF16, w=ODD), _lib.LK_EINVAL), (dict(out=ODD), _lib.LK_EINVAL),
    (dict(bias=ODD), _lib.LK_EINVAL), (dict(sa=ODD), _lib.LK_EINVAL), (dict(sw=ODD), _lib.LK_EINVAL), (dict(r=ODD, ldr=4), _lib.LK_EINVAL),
    (dict(device=-1), _lib.LK_ECUDA),
])
def test_linear_refuses(kw, status):
    assert linear(**kw) == status
    assert b"lk_linear" in _lib.lib.lk_last_error()


def sample(**kw):
    a = dict(device=0, dtype=F32, rows=4, vocab=8, x=P, ld=8, t=None, k=None, p=None, mp=None, u=P, ids=P, probs=P, kept=P, st=None)
    a.update(kw)
    return _lib.lib.lk_sample(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=I8), _lib.LK_EINVAL), (dict(rows=-1), _lib.LK_EINVAL), (dict(vocab=-1), _lib.LK_EINVAL),
    (dict(vocab=(1 << 24) + 1, ld=1 << 25), _lib.LK_ERANGE), (dict(rows=1 << 31), _lib.LK_ERANGE),
    (dict(x=None), _lib.LK_EINVAL), (dict(u=None), _lib.LK_EINVAL), (dict(ids=None), _lib.LK_EINVAL), (dict(ld=7), _lib.LK_EINVAL),
    (dict(x=ODD), _lib.LK_EINVAL), (dict(t=ODD), _lib.LK_EINVAL), (dict(k=ODD), _lib.LK_EINVAL), (dict(p=ODD), _lib.LK_EINVAL),
    (dict(mp=ODD), _lib.LK_EINVAL), (dict(u=ODD), _lib.LK_EINVAL), (dict(ids=C.c_void_p(4100)), _lib.LK_EINVAL),
    (dict(probs=ODD), _lib.LK_EINVAL), (dict(kept=ODD), _lib.LK_EINVAL), (dict(device=-1), _lib.LK_ECUDA),
])
def test_sample_refuses(kw, status):
    assert sample(**kw) == status
    assert b"lk_sample" in _lib.lib.lk_last_error()


def test_no_cpu_fallback():
    x = torch.zeros(2, 16)
    for call in (lambda: ops.rms_norm_i8(x), lambda: ops.linear(x.to(torch.int8), x.to(torch.int8)), lambda: ops.sample(x, torch.zeros(2))):
        with pytest.raises(_lib.LokiError, match="CUDA tensor"):
            call()
    if _lib.device_count() == 0:
        assert norm() == linear() == sample() == _lib.LK_ECUDA
        assert b"no CPU path" in _lib.lib.lk_last_error()


def test_bfloat16_is_no_storage_type():
    h = C.c_void_p()
    assert _lib.lib.lk_index_create(8, BF16, 0, 0, C.byref(h)) == _lib.LK_EINVAL
