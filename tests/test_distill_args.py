"""What the top logits and the distillation refuse, on the host: no call here
reaches the GPU."""
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

    return _lib.DistillShape(**{**dict(n=10, C=20, K=4, dtype=0, valueDtype=0, idBytes=4, reduction=1, temperature=1.0), **k})


def test_python_refuses_what_is_not_on_the_device():
    from tcc_amd import training

    z, v, i = torch.zeros((4, 6)), torch.zeros((4, 2)), torch.zeros((4, 2), dtype=torch.int32)
    for call in (lambda: training.top_logits(z, 2), lambda: training.distill_loss(z, v, i),
                 lambda: training.distill_grad(z[0, 0], z, v, i, torch.zeros((4, 4)))):
        with pytest.raises(TypeError):
            call()


def test_top_logits_refusals():
    L = lib()
    call = lambda **k: L.tcc_top_logits(*{**dict(z=P, ldz=20, dt=0, n=10, C=20, K=4, t=1.0, v=P, ldv=4, i=P, ldi=4, r=P,  # noqa: E731
                                                 st=None), **k}.values())
    for k in (dict(dt=3), dict(K=0), dict(K=21), dict(t=0.0), dict(t=-1.0), dict(t=float("nan")), dict(t=float("inf")),
              dict(z=None), dict(v=None), dict(i=None), dict(ldz=19), dict(ldv=3), dict(ldi=3)):
        assert call(**k) == INVALID, k
    assert b"top logits" in L.tcc_last_error()
    assert call(C=100, ldz=100, K=65, ldv=65, ldi=65) == UNSUPPORTED
    assert call(C=1 << 31, ldz=1 << 31) == UNSUPPORTED and call(n=1 << 40) == UNSUPPORTED
    assert call(n=0, z=None) == 0  # nothing to do


def test_distillation_refusals():
    L = lib()

    def loss(s, **k):
        a = {**dict(z=P, ldz=20, v=P, ldv=4, i=P, ldi=4, rest=None, w=None, loss=P, total=None, stats=P, err=None, ws=P,
                    bytes=1 << 20, st=None), **k}
        return L.tcc_distill_loss(ctypes.byref(s), *a.values())

    def grad(s, **k):
        a = {**dict(dl=P, z=P, ldz=20, v=P, ldv=4, i=P, ldi=4, rest=None, w=None, total=None, stats=P, dz=P, ldd=20, st=None),
             **k}
        return L.tcc_distill_grad(ctypes.byref(s), *a.values())

    for k in (dict(C=0), dict(K=0), dict(dtype=3), dict(valueDtype=3), dict(idBytes=2), dict(reduction=3),
              dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=float("inf"))):
        assert loss(shape(**k)) == INVALID and grad(shape(**k)) == INVALID, k
        assert L.tcc_distill_loss_workspace_bytes(ctypes.byref(shape(**k))) == 0
    for k in (dict(K=65), dict(C=1 << 31), dict(n=1 << 40)):
        s = shape(**k)
        big = dict(ldz=1 << 31, ldv=65, ldi=65)
        assert loss(s, **big) == UNSUPPORTED and grad(s, **big, ldd=1 << 31) == UNSUPPORTED, k
    for k in (dict(z=None), dict(v=None), dict(i=None), dict(stats=None), dict(ldz=19), dict(ldv=3), dict(ldi=3),
              dict(stats=ctypes.c_void_p(72))):
        assert loss(shape(), **k) == INVALID and grad(shape(), **k) == INVALID, k
    for k in (dict(loss=None), dict(ws=None), dict(bytes=8), dict(ws=ctypes.c_void_p(72))):
        assert loss(shape(), **k) == INVALID, k
    for k in (dict(dl=None), dict(dz=None), dict(ldd=19), dict(w=P), dict(total=P)):
        assert grad(shape(), **k) == INVALID, k
    assert loss(shape(n=0, reduction=0), loss=None) == 0 and grad(shape(n=0)) == 0  # nothing to do


def test_temperatures_without_a_finite_inverse_or_square_are_refused():
    L = lib()
    for t in (1e-19, 1e-40, 2e18):
        assert L.tcc_top_logits(P, 20, 0, 10, 20, 4, t, P, 4, P, 4, P, None) == INVALID
        s = shape(temperature=t)
        assert L.tcc_distill_loss(ctypes.byref(s), P, 20, P, 4, P, 4, None, None, P, None, P, None, P, 1 << 20, None) == INVALID
        assert L.tcc_distill_grad(ctypes.byref(s), P, P, 20, P, 4, P, 4, None, None, None, P, P, 20, None) == INVALID
