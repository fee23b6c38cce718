"""The global gradient norm, clipping and the Adam step (tcc_amd.training)
against plain 64-bit evaluations.

The norm is summed in 64 bits and rounded once, and its factor takes a sum
and a quotient in fp32: 4 u of itself, u = 2^-24.  A clipped gradient adds
its product and the rounding to its type.  The Adam step's moments are off by
a few u of their terms, the step by a few u of itself (quotients, a square
root) and by what the moments are off; 16 u covers their sum."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
U_OUT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1,), (7,), (100, 256), (256,), (256, 2), (3, 5, 11), (8192,), (4097,), (20_011, 3), (0, 4)]


def tensors(shapes, types, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=gen) * scale).to(types[i % len(types)]).cuda() for i, s in enumerate(shapes)]


def norm64(grads):
    return float(np.sqrt(sum(float((g.double().cpu() ** 2).sum()) for g in grads)))


def floor_of(t):  # half the distance of fp16's smallest values
    return 2.0**-25 if t == torch.float16 else 0.0


def check_clipped(out, before, norm, max_norm):
    total = norm64(before)
    assert abs(float(norm) - total) <= 2 * U * total
    c = min(1.0, max_norm / (total + 1e-6))
    for o, g in zip(out, before):
        want = g.double().cpu() * c
        tol = (5 * U + U_OUT[o.dtype]) * want.abs() * 1.01 + floor_of(o.dtype)
        assert bool(((o.double().cpu() - want).abs() <= tol).all())


@pytest.mark.parametrize("types", [[t] for t in TYPES] + [TYPES])
@pytest.mark.parametrize("max_norm", [0.5, 3.0, 1e9])
def test_clip(gpu, types, max_norm):
    from tcc_amd import training

    grads = tensors(SHAPES, types, 1)
    before = [g.clone() for g in grads]
    out = [torch.full_like(g, 9.0) for g in grads]
    n1 = training.clip_grad_norm(grads, max_norm, out=out)
    assert all(torch.equal(a, b) for a, b in zip(grads, before)), "the gradients stay where out is given"
    check_clipped(out, before, n1, max_norm)
    n2 = training.clip_grad_norm(grads, max_norm)
    assert torch.equal(n1, n2) and all(torch.equal(a, b) for a, b in zip(grads, out))
    assert torch.equal(training.grad_norm(before), n1)
    if max_norm == 1e9:
        assert all(torch.equal(a, b) for a, b in zip(grads, before)), "below the largest norm nothing changes"


@pytest.mark.parametrize("count", [0, 1, 58, 59, 60, 119, 300])
def test_long_lists(gpu, count):
    """Lists beyond what one launch's arguments hold, empty ones among them."""
    from tcc_amd import training

    grads = tensors([(k % 5, 3 + k) for k in range(count)], TYPES, count)
    before = [g.clone() for g in grads]
    norm = training.clip_grad_norm(grads, 1.0)
    check_clipped(grads, before, norm, 1.0)
    check_adam(tensors([g.shape for g in grads], [torch.float32], 7), before, 1.0, True, 0.01)


def test_strided_tensors(gpu):
    """Rows of a wider buffer, transposed weights and odd addresses, in place
    and beside contiguous outputs; the buffer around them stays."""
    from tcc_amd import training

    room = torch.randn((300, 128), device="cuda")
    kept = room.clone()
    grads = [room[:, 5:70], room[10:20, 100:101], torch.randn((64, 33), device="cuda").t(),
             torch.randn(1001, device="cuda")[1:], torch.randn((2, 6, 40), device="cuda")[:, :, 8:24]]
    before = [g.clone() for g in grads]
    out = [torch.empty_like(g) for g in before]
    check_clipped(out, before, training.clip_grad_norm(grads, 2.0, out=out), 2.0)
    check_clipped(grads, before, training.clip_grad_norm(grads, 2.0), 2.0)
    outside = torch.ones_like(room, dtype=torch.bool)
    outside[:, 5:70] = False
    outside[10:20, 100] = False
    assert torch.equal(room[outside], kept[outside])
    with pytest.raises(ValueError):  # three strides of their own
        training.grad_norm([torch.randn((4, 6, 10), device="cuda")[:, ::2, ::2]])
    with pytest.raises(ValueError):  # overlapping elements
        training.clip_grad_norm([torch.randn((1, 5), device="cuda").expand(4, 5)], 1.0)


def test_norms_of_extreme_values(gpu):
    """Squares that leave fp32's range, and norms that are no numbers."""
    from tcc_amd import training

    g = torch.full((1000,), 1e30, device="cuda")
    assert abs(float(training.grad_norm([g])) - 1e30 * 1000**0.5) <= 1e24 * 10
    g.fill_(1e-30)
    assert abs(float(training.grad_norm([g])) - 1e-30 * 1000**0.5) <= 1e-36 * 10
    g[7] = float("inf")
    other = torch.ones(5, device="cuda")
    norm = training.clip_grad_norm([g, other], 1.0)
    assert float(norm) == float("inf") and bool((other == 0).all()) and bool(g[7].isnan())
    other.fill_(1.0)
    other[2] = float("nan")
    third = torch.ones(5, device="cuda")
    assert bool(training.clip_grad_norm([other, third], 1.0).isnan()) and bool(third.isnan().all())
    zero = torch.zeros(9, device="cuda")
    assert float(training.clip_grad_norm([zero], 1.0)) == 0.0 and bool((zero == 0).all())
    ones = torch.ones(9, device="cuda")
    training.clip_grad_norm([ones], 0.0)
    assert bool((ones == 0).all())


def adam64(p, g, m, v, t, c, lr, betas, eps, wd, decoupled):
    b1, b2 = betas
    g = g * c + (0.0 if decoupled else wd) * p
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    step = lr / (1 - b1**t) * m2 / (np.sqrt(v2) / np.sqrt(1 - b2**t) + eps)
    keep = 1 - lr * wd if decoupled else 1.0
    near_m = 16 * U * (b1 * np.abs(m) + (1 - b1) * (np.abs(g) + np.abs(p) * wd))
    near = 16 * U * np.abs(step) + lr / (1 - b1**t) * near_m / (np.sqrt(v2) / np.sqrt(1 - b2**t) + eps)
    return keep * p - step, m2, v2, near + 4 * U * np.abs(p), near_m


def check_adam(params, grads, max_norm, decoupled, wd, lr=3e-3, betas=(0.9, 0.999), eps=1e-8, start=4):
    from tcc_amd import training

    m = tensors([p.shape for p in params], [torch.float32], 50, 0.1)
    v = [x.square() for x in tensors([p.shape for p in params], [torch.float32], 60, 0.1)]
    step = torch.tensor(start, dtype=torch.int64, device="cuda")
    old = [[x.double().cpu().numpy() for x in xs] for xs in (params, grads, m, v)]
    kept = [g.clone() for g in grads]
    norm = training.adam_step(params, grads, m, v, step, lr=lr, betas=betas, eps=eps, weight_decay=wd,
                              decoupled=decoupled, max_norm=max_norm)
    assert int(step) == start + 1
    assert all(torch.equal(a, b) for a, b in zip(grads, kept))
    total = norm64(grads)
    assert (norm is None) == (max_norm is None)
    c = 1.0 if max_norm is None else min(1.0, max_norm / (total + 1e-6))
    if norm is not None:
        assert abs(float(norm) - total) <= 2 * U * total
    for i, p in enumerate(params):
        want, m2, v2, near, near_m = adam64(*(o[i] for o in old), start + 1, c, lr, betas, eps, wd, decoupled)
        got = p.double().cpu().numpy()
        assert np.all(np.abs(got - want) <= near + U_OUT[p.dtype] * np.abs(want) * 1.01 + floor_of(p.dtype))
        assert np.all(np.abs(m[i].double().cpu().numpy() - m2) <= near_m)
        assert np.all(np.abs(v[i].double().cpu().numpy() - v2) <= 16 * U * v2 + 1e-37)


@pytest.mark.parametrize("ptypes,gtypes", [([torch.float32], [torch.float32]), ([torch.bfloat16], [torch.bfloat16]),
                                           (TYPES, [torch.bfloat16, torch.float32])])
@pytest.mark.parametrize("max_norm,decoupled,wd", [(None, True, 0.0), (1.0, True, 0.01), (2.0, False, 0.1), (1e9, False, 0.0)])
def test_adam(gpu, ptypes, gtypes, max_norm, decoupled, wd):
    check_adam(tensors(SHAPES, ptypes, 2), tensors(SHAPES, gtypes, 3), max_norm, decoupled, wd)


def test_adam_first_step_from_zero_moments(gpu):
    from tcc_amd import training

    p, g = tensors([(33, 5)], [torch.float32], 4), tensors([(33, 5)], [torch.float32], 5)
    g[0][0] = 0.0  # no gradient and no moment: 0 / (0 + eps)
    m, v = [torch.zeros_like(p[0])], [torch.zeros_like(p[0])]
    step = torch.zeros((), dtype=torch.int64, device="cuda")
    q = [p[0].clone().requires_grad_(True)]
    q[0].grad = g[0].clone()
    opt = torch.optim.AdamW(q, lr=0.01, weight_decay=0.1)
    opt.step()
    training.adam_step(p, g, m, v, step, lr=0.01, weight_decay=0.1)
    assert bool(((p[0] - q[0]).abs() <= 32 * U * (q[0].abs() + 0.01)).all()) and bool(torch.isfinite(p[0]).all())


def test_adam_strided(gpu):
    """A parameter that is rows of a wider buffer, and a transposed one."""
    room = torch.randn((50, 64), device="cuda")
    params = [room[:, 3:40], torch.randn((30, 20), device="cuda").t(), torch.randn(77, device="cuda")[1:]]
    kept = room.clone()
    grads = tensors([(50, 37)], [torch.float32], 6) + [torch.randn((30, 20), device="cuda").t(),
                                                       torch.randn(76, device="cuda")]
    from tcc_amd import training

    same = [torch.zeros((50, 37), device="cuda"), torch.zeros((30, 20), device="cuda").t(), torch.zeros(76, device="cuda")]
    m, v = [x.clone() for x in same], [x.clone() for x in same]
    want = [p.clone().contiguous() for p in params]
    wm, wv = [x.contiguous() for x in same], [x.clone().contiguous() for x in same]
    s1, s2 = (torch.zeros((), dtype=torch.int64, device="cuda") for _ in range(2))
    training.adam_step(params, grads, m, v, s1, max_norm=1.0)
    training.adam_step(want, [g.contiguous() for g in grads], wm, wv, s2, max_norm=1.0)
    assert all(torch.equal(a, b) for a, b in zip(params + m + v, want + wm + wv))
    assert torch.equal(room[:, :3], kept[:, :3]) and torch.equal(room[:, 40:], kept[:, 40:])


def test_places_past_32_bits(gpu):
    """A gradient of rows that lie over 2^32 elements apart, and one of more
    elements than 32 bits count."""
    from tcc_amd import training

    room = torch.zeros((3, 2_200_000_000), dtype=torch.bfloat16, device="cuda")
    room[2, 1:6] = 3.0
    room[0, 1:6] = 4.0
    norm = training.clip_grad_norm([room[:, :7]], 1.0)
    assert abs(float(norm) - (5 * 25) ** 0.5) <= 1e-6
    assert abs(float(room[2, 3]) - 3.0 / 125**0.5) <= 2.0**-8
    room[2, -1] = 2.0  # the whole buffer, as one run
    before = float(training.grad_norm([room]))
    assert abs(float(training.clip_grad_norm([room], before / 2)) - before) <= 1e-6
    assert abs(float(room[2, -1]) - 1.0) <= 2.0**-7


def test_replayed_graph_and_other_stream(gpu):
    from tcc_amd import training

    p, g = tensors(SHAPES, [torch.float32], 8), tensors(SHAPES, [torch.float32], 9)
    m, v = [torch.zeros_like(x) for x in p], [torch.zeros_like(x) for x in p]
    step = torch.zeros((), dtype=torch.int64, device="cuda")
    twin = [[x.clone() for x in xs] for xs in (p, m, v)]
    twin_step = step.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    n1 = training.adam_step(p, g, m, v, step, max_norm=1.0, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    n2 = training.adam_step(twin[0], g, twin[1], twin[2], twin_step, max_norm=1.0)
    assert torch.equal(n1, n2) and all(torch.equal(a, b) for a, b in zip(p, twin[0]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = training.adam_step(p, g, m, v, step, max_norm=1.0)
    for k in range(3):
        for x in g:
            x.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = training.adam_step(twin[0], g, twin[1], twin[2], twin_step, max_norm=1.0)
        assert torch.equal(norm, want) and int(step) == int(twin_step) == k + 2
        assert all(torch.equal(a, b) for a, b in zip(p + m + v, twin[0] + twin[1] + twin[2]))


@pytest.mark.parametrize("decoupled,decay", [(True, 0.1), (True, 0.0), (False, 0.0)])
@pytest.mark.parametrize("n", [5, 5000])
def test_infinite_parameters_leave_the_moments(gpu, decoupled, decay, n):
    """The gradient holds no parameter unless its decay does: the moments stay
    those of the gradients beside an infinite or NaN parameter."""
    from tcc_amd import training

    p, g = tensors([(n,)], [torch.float32], 3)[0], tensors([(n,)], [torch.float32], 4)[0]
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    p[0], p[3] = float("inf"), float("nan")
    training.adam_step([p], [g], [m], [v], torch.zeros((), dtype=torch.int64, device="cuda"), weight_decay=decay,
                       decoupled=decoupled)
    assert bool(p[0].isinf()) and bool(p[3].isnan()) and int(p.isfinite().sum()) == n - 2
    assert bool(((m - 0.1 * g).abs() <= 4 * U * g.abs()).all())
    assert bool(((v - 0.001 * g * g).abs() <= 8 * U * g * g).all())
