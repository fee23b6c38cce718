"""What tcc_amd.training and include/tcc_training.h refuse, on the host: no
call here reaches the GPU."""
import ctypes

import pytest
import torch

INVALID, UNSUPPORTED = 1, 3
P = ctypes.c_void_p(64)  # an address that is never read


def lib():
    from tcc_amd import _lib

    return _lib.lib()


def test_python_refuses_what_is_not_on_the_device():
    from tcc_amd import training

    x, ids = torch.zeros((4, 6)), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: training.embedding_lookup(x, ids),
                 lambda: training.embedding_grad(x, ids, 9),
                 lambda: training.group_norm(x, 2),
                 lambda: training.group_norm_grad(x, x, x, x, 2),
                 lambda: training.grad_norm([x]),
                 lambda: training.clip_grad_norm([x], 1.0),
                 lambda: training.adam_step([x], [x], [x], [x], torch.zeros((), dtype=torch.int64))):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(TypeError):
        training.grad_norm([torch.zeros(3, dtype=torch.float64)])


def test_python_refuses_values():
    from tcc_amd import training

    x = torch.zeros((4, 6))
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            training.clip_grad_norm([x], bad)
    with pytest.raises(ValueError):
        training.clip_grad_norm([x], 1.0, out=[x.half()])


def test_embedding_refusals():
    L = lib()
    look = lambda **k: L.tcc_embedding_lookup(*{**dict(t=P, ldt=8, dt=0, ids=P, ib=4, n=3, V=5, D=8, s=1.0, pad=-1,  # noqa: E731
                                                       out=P, ldo=8, err=None, st=None), **k}.values())
    for k in (dict(dt=3), dict(ib=2), dict(ids=None), dict(D=0), dict(ldt=7), dict(ldo=7), dict(t=None), dict(out=None)):
        assert look(**k) == INVALID, k
    assert b"embedding" in L.tcc_last_error()
    assert look(n=0xFFFFFFFF) == UNSUPPORTED and look(V=1 << 40) == UNSUPPORTED
    assert look(n=0) == 0  # nothing to do
    grad = lambda **k: L.tcc_embedding_grad(*{**dict(d=P, ldd=8, dt=0, ids=P, ib=4, n=3, V=5, D=8, s=1.0, pad=-1, g=P,  # noqa: E731
                                                     ldg=8, acc=0, err=None, ws=P, bytes=1 << 20, st=None), **k}.values())
    for k in (dict(dt=9), dict(ib=1), dict(ldd=7), dict(ldg=7), dict(d=None), dict(g=None), dict(ws=None), dict(bytes=8),
              dict(ws=ctypes.c_void_p(68))):
        assert grad(**k) == INVALID, k
    assert grad(n=0, acc=1) == 0
    assert L.tcc_embedding_grad_workspace_bytes(1000, 4096, 32) >= 16 * 1000


def test_group_norm_refusals():
    from tcc_amd import _lib

    L = lib()

    def shape(**k):
        return _lib.GroupNormShape(**{**dict(N=10, B=2, maxRows=0, C=8, G=2, offsets=None, offsetBytes=0, dtype=0,
                                             paramDtype=0, activation=0, eps=1e-5), **k})

    def call(s, **k):
        a = {**dict(x=P, ldx=8, w=None, b=None, y=P, ldy=8, mean=P, rstd=P, ws=P, bytes=1 << 24, st=None), **k}
        return L.tcc_group_norm(ctypes.byref(s), *a.values())

    for k in (dict(G=0), dict(G=3), dict(C=0), dict(dtype=7), dict(paramDtype=7), dict(activation=4), dict(N=9),
              dict(B=0), dict(eps=-1.0), dict(eps=float("nan")), dict(offsets=64, offsetBytes=2),
              dict(offsets=64, offsetBytes=4, B=0)):
        s = shape(**k)
        assert call(s) == INVALID, k
        assert L.tcc_group_norm_workspace_bytes(ctypes.byref(s), 1) == 0
    assert call(shape(C=8192, G=2), ldx=8192, ldy=8192) == UNSUPPORTED
    for k in (dict(x=None), dict(y=None), dict(ldx=7), dict(ldy=7), dict(mean=None), dict(rstd=None), dict(ws=None),
              dict(bytes=4), dict(ws=ctypes.c_void_p(72))):
        assert call(shape(), **k) == INVALID, k
    assert L.tcc_group_norm(None, P, 8, None, None, P, 8, P, P, P, 1 << 20, None) == INVALID
    g = lambda s, **k: L.tcc_group_norm_grad(ctypes.byref(s), *{**dict(d=P, ldd=8, x=P, ldx=8, mean=P, rstd=P, w=None,  # noqa: E731
                                                                       b=None, dx=P, lddx=8, dw=None, db=None, ws=P,
                                                                       bytes=1 << 24, st=None), **k}.values())
    for k in (dict(d=None), dict(x=None), dict(dx=None), dict(ldd=7), dict(ldx=7), dict(lddx=7), dict(mean=None),
              dict(rstd=None), dict(ws=None), dict(bytes=4)):
        assert g(shape(), **k) == INVALID, k


def test_list_refusals():
    from tcc_amd import _lib

    L = lib()

    def arr(*tensors):
        flat = [v for t in tensors for v in t]
        return (ctypes.c_uint64 * max(len(flat), 1))(*flat)

    good = arr((64, 1, 10, 10, 0))
    need = L.tcc_grad_norm_workspace_bytes()
    for bad in (arr((64, 1, 10, 10, 3)), arr((0, 1, 10, 10, 0)), arr((64, 2, 10, 9, 0))):
        assert L.tcc_grad_norm(bad, 1, P, P, need, None) == INVALID
    assert L.tcc_grad_norm(arr((64, 1 << 40, 1 << 20, 1 << 20, 0)), 1, P, P, need, None) == UNSUPPORTED
    assert L.tcc_grad_norm(None, 1, P, P, need, None) == INVALID
    assert L.tcc_grad_norm(good, 1, None, P, need, None) == INVALID
    assert L.tcc_grad_norm(good, 1, P, P, need - 1, None) == INVALID
    assert L.tcc_grad_norm(good, 1, P, ctypes.c_void_p(72), need, None) == INVALID
    for out in (arr((64, 2, 5, 5, 0)), arr((64, 1, 10, 10, 1))):
        assert L.tcc_clip_grad_norm(good, out, 1, 1.0, P, P, need, None) == INVALID
    for norm in (-1.0, float("nan")):
        assert L.tcc_clip_grad_norm(good, good, 1, norm, P, P, need, None) == INVALID
    half = arr((64, 1, 10, 10, 2))
    for k in (dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0)):
        a = _lib.Adam(**{**dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weightDecay=0.0, maxNorm=-1.0, decoupled=1), **k})
        assert L.tcc_adam_step(good, good, good, good, 1, ctypes.byref(a), P, P, P, need, None) == INVALID, k
    a = _lib.Adam(1e-3, 0.9, 0.99, 1e-8, 0.0, -1.0, 1)
    assert L.tcc_adam_step(good, good, half, good, 1, ctypes.byref(a), P, P, P, need, None) == INVALID
    assert L.tcc_adam_step(good, good, good, good, 1, ctypes.byref(a), None, P, P, need, None) == INVALID
    assert L.tcc_adam_step(good, good, good, good, 1, None, P, P, P, need, None) == INVALID


def test_optimizer_takes_one_group():
    from tcc_amd import gcn

    first, second = (torch.nn.Parameter(torch.zeros(3)) for _ in range(2))
    with pytest.raises(ValueError):
        gcn.ClippedAdam([{"params": [first]}, {"params": [second]}])
    optimizer = gcn.ClippedAdam([first])
    with pytest.raises(ValueError):  # later too: step() would pass over it
        optimizer.add_param_group({"params": [second]})
    assert len(optimizer.param_groups) == 1


def test_embedding_moves_as_a_whole():
    """The error word goes where the table goes, and is in no checkpoint."""
    from tcc_amd import gcn

    e = gcn.NodeEmbedding(6, 4, device="cpu")
    assert list(e.state_dict()) == ["weight"]
    e = e.to("meta").to(torch.bfloat16)
    assert e.weight.dtype == torch.bfloat16
    assert e.device_error.device.type == "meta" and e.device_error.dtype == torch.int32


def test_rows_too_wide_are_refused():
    """Column counts that the kernels' 32-bit arithmetic does not hold."""
    L = lib()
    for D in (0xFFFFFFFF, 0xFFFFFFFF - 100):
        assert L.tcc_embedding_lookup(P, D, 1, P, 4, 3, 5, D, 1.0, -1, ctypes.c_void_p(66), D, None, None) == UNSUPPORTED
    for D in (1 << 28, 0xFFFFFFFF):
        assert L.tcc_embedding_grad(P, D, 0, P, 4, 3, 5, D, 1.0, -1, P, D, 0, None, P, 1 << 40, None) == UNSUPPORTED
