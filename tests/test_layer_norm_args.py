"""What the layer norm refuses, on the host: no call here reaches the GPU."""
import ctypes

import pytest
import torch

INVALID, UNSUPPORTED = 1, 3
P = ctypes.c_void_p(64)  # an address that is never read


def lib():
    from tcc_amd import _lib

    return _lib.lib()


def shape(**k):
    from tcc_amd import _lib

    return _lib.LayerNormShape(**{**dict(N=10, C=8, dtype=0, paramDtype=0, activation=0, eps=1e-5), **k})


def test_python_refuses_what_is_not_on_the_device():
    from tcc_amd import training

    x, s = torch.zeros((4, 6)), torch.zeros(4)
    for call in (lambda: training.layer_norm(x), lambda: training.layer_norm_grad(x, x, s, s)):
        with pytest.raises(TypeError):
            call()


def test_layer_norm_refusals():
    L = lib()
    call = lambda s, **k: L.tcc_layer_norm(ctypes.byref(s), *{**dict(x=P, ldx=8, res=None, ldr=0, w=None, b=None, y=P, ldy=8,  # noqa: E731
                                                                     sum=None, lds=0, mean=P, rstd=P, st=None), **k}.values())
    for k in (dict(C=0), dict(dtype=3), dict(paramDtype=7), dict(activation=4), dict(eps=-1.0), dict(eps=float("nan"))):
        assert call(shape(**k)) == INVALID, k
        assert L.tcc_layer_norm_grad_workspace_bytes(ctypes.byref(shape(**k))) == 0
    assert b"layer norm" in L.tcc_last_error()
    assert call(shape(C=16385), ldx=16385, ldy=16385) == UNSUPPORTED
    assert call(shape(N=1 << 40)) == UNSUPPORTED
    for k in (dict(x=None), dict(y=None), dict(ldx=7), dict(ldy=7), dict(mean=None), dict(rstd=None), dict(res=P, ldr=7),
              dict(sum=P, lds=7)):
        assert call(shape(), **k) == INVALID, k
    assert L.tcc_layer_norm(None, P, 8, None, 0, None, None, P, 8, None, 0, P, P, None) == INVALID
    assert call(shape(N=0), x=None, y=None) == 0  # nothing to do


def test_layer_norm_gradient_refusals():
    L = lib()
    call = lambda s, **k: L.tcc_layer_norm_grad(ctypes.byref(s), *{**dict(  # noqa: E731
        d=P, ldd=8, h=P, ldh=8, mean=P, rstd=P, w=None, b=None, add=None, lda=0, dx=P, lddx=8, dw=P, db=None, ws=P,
        bytes=1 << 24, st=None), **k}.values())
    for k in (dict(C=0), dict(dtype=9), dict(activation=17)):
        assert call(shape(**k)) == INVALID, k
    assert call(shape(C=20000), ldd=20000, ldh=20000, lddx=20000) == UNSUPPORTED
    for k in (dict(d=None), dict(h=None), dict(dx=None), dict(ldd=7), dict(ldh=7), dict(lddx=7), dict(mean=None),
              dict(rstd=None), dict(add=P, lda=7), dict(ws=None), dict(bytes=4), dict(ws=ctypes.c_void_p(72))):
        assert call(shape(), **k) == INVALID, k
    assert L.tcc_layer_norm_grad(None, P, 8, P, 8, P, P, None, None, None, 0, P, 8, P, P, P, 1 << 24, None) == INVALID
    assert call(shape(N=0), d=None, h=None, dx=None, dw=None) == 0  # no rows, no sums
