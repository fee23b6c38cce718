"""The distillation loss against a teacher's entries and its gradient
(tcc_amd.training), against plain 64-bit evaluations.

Bounds, with u = 2^-24 and x = (z - m) / T: an exponent has three roundings, and
the mean of |x| over the shares is at most log C, so that a sum s of C shares is
off by 3 u log C of itself, and by C / 64 + 100 roundings of its additions over
4 lanes (16 vectors of up to 8 each, few classes) to 256: E = (C / 64 + 300) u
for all of it, teacher's sums too.  A row's loss is T^2 sum p (log p - log q):
E (1 + |log p - log q|) for each p, and 8 u of the logarithms, which are
differences of what has been rounded.  A gradient is a difference of
probabilities, each off by E + 4 u |x| of itself, and one rounding to its type."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
U_OUT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 1e-30, torch.bfloat16: 1e-30, torch.float16: 2.0**-25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1, 1), (5, 2, 2), (7, 3, 1), (64, 7, 7), (30, 6, 40), (40, 8, 3), (300, 47, 4), (101, 100, 8), (33, 257, 64),
          (200, 64, 16), (50, 129, 17), (20, 1000, 33), (9, 4096, 64), (7, 4097, 5), (5, 50_001, 32), (3, 140_000, 64),
          (2, 262_150, 64)]


def inputs(n, C, K, dtype, seed, ids_type=torch.int32, value_type=None, spread=3.0, some_absent=True):
    """A teacher's entries (distinct where there are classes enough, some of them
    absent, some rows without any) and a student that follows it."""
    gen = torch.Generator().manual_seed(seed)
    t = torch.randn((n, C), generator=gen) * spread
    if K <= C:
        values, ids = torch.topk(t, K, dim=1)
    else:
        ids = torch.randint(0, C, (n, K), generator=gen)
        values = t.gather(1, ids)
    if some_absent and n > 1:
        ids[torch.rand((n, K), generator=gen) < 0.1] = -1
        ids[n // 2] = -1
        values[n // 3, 0] = -np.inf
    z = (0.7 * t + torch.randn((n, C), generator=gen)).to(dtype).cuda()
    rest = torch.randn(n, generator=gen).cuda()
    w = (torch.rand(n, generator=gen) + 0.1) * (torch.rand(n, generator=gen) < 0.8)
    return z, values.to(value_type or dtype).cuda(), ids.to(ids_type).cuda(), rest, w.cuda()


def exact(z, values, ids, rest, T, w, reduction):
    """(loss, its tolerance, gradient, its tolerance), in 64 bits on the CPU; the
    gradient from a d_loss of 1."""
    n, C = z.shape
    z, t, ids = z.double().cpu(), values.double().cpu(), ids.cpu().long()
    w = torch.ones(n, dtype=torch.float64) if w is None else w.double().cpu()
    there = (ids >= 0) & (ids < C)
    safe = torch.where(there, ids, 0)
    t = torch.where(there, t, -np.inf)
    picked = torch.zeros((n, C), dtype=torch.bool)
    picked.view(-1)[(torch.arange(n)[:, None] * C + safe)[there]] = True
    log_q = torch.log_softmax(z / T, 1)
    x = ((z - z.amax(1, keepdim=True)) / T).clamp(min=-1e4)  # -inf has no share
    at = log_q.gather(1, safe)
    xs = x.gather(1, safe)
    if rest is not None:
        t = torch.cat([t, rest.double().cpu()[:, None]], 1)
        others = torch.logsumexp(log_q.masked_fill(picked, -np.inf), 1, keepdim=True)
        at = torch.cat([at, others], 1)
        xs = torch.cat([xs, torch.zeros((n, 1))], 1)
    some = (t > -np.inf).any(1) & (w != 0)
    log_p = torch.log_softmax(torch.where(some[:, None], t, 0.0) / T, 1)
    p = torch.where(some[:, None], log_p.exp(), 0.0)
    E = (C / 64 + 300) * U
    term = lambda v: torch.where(p > 0, p * v, 0.0).sum(1)  # noqa: E731
    rows = T * T * w * term(log_p - at)
    tol = T * T * w * term(E * (1 + (log_p - at).abs()) + 8 * U * (log_p.abs() + at.abs() + xs.abs()))
    rows, tol = torch.where(some, rows, 0.0), torch.where(some, tol, 0.0)
    scale = w if reduction != "mean" else w / (w.sum() if w.sum() != 0 else 1.0)
    if reduction != "none":
        by = w.sum() if reduction == "mean" and w.sum() != 0 else 1.0
        rows, tol = rows.sum() / by, tol.sum() / abs(by)
    K = ids.shape[1]
    aim = torch.zeros((n, C), dtype=torch.float64).scatter_add_(1, safe, torch.where(there, p[:, :K], 0.0))
    q = log_q.exp()
    size = q + aim
    if rest is not None:
        spread = torch.where(picked, 0.0, (log_q - others).exp() * p[:, K:])
        aim, size = aim + spread, size + spread
    g = T * (scale * some)[:, None]
    grad = torch.where(g != 0, g * (q - aim), 0.0)
    gtol = torch.where(g != 0, g.abs() * size * (E + 4 * U * x.abs()), 0.0)
    return rows, tol + U * rows.abs() + 1e-30, grad, gtol


def check(z, values, ids, rest=None, T=1.0, w=None, reduction="mean", error=None):
    from tcc_amd import training

    loss, stats, total = training.distill_loss(z, values, ids, rest=rest, temperature=T, weight=w, reduction=reduction,
                                               device_error=error)
    rows, tol, grad, gtol = exact(z, values, ids, rest, T, w, reduction)
    assert loss.shape == rows.shape and stats.shape == (z.shape[0], 4)
    # a rest of which the student has nothing, all classes being entries, is an infinite loss
    err = torch.where(loss.cpu() == rows, 0.0, (loss.double().cpu() - rows).abs())
    assert bool((err <= tol).all()), f"loss: largest excess {float((err - tol).max()):.3e}"
    d_loss = torch.full(loss.shape, 0.75, device="cuda")
    back = lambda: training.distill_grad(d_loss, z, values, ids, stats, rest=rest, temperature=T, weight=w, total=total,  # noqa: E731
                                         reduction=reduction)
    dz = back()
    assert dz.dtype == z.dtype
    want, gtol = 0.75 * grad, 0.75 * gtol
    gtol = gtol + U_OUT[z.dtype] * (want.abs() + gtol) + TINY[z.dtype]
    err = (dz.double().cpu() - want).abs()
    assert bool((err <= gtol).all()), f"gradient: largest excess {float((err - gtol).max()):.3e}"
    again = training.distill_loss(z, values, ids, rest=rest, temperature=T, weight=w, reduction=reduction)
    assert torch.equal(loss, again[0]) and torch.equal(stats, again[1]) and torch.equal(dz, back()), "the same bits"
    return loss, dz


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,C,K", SHAPES)
def test_both_passes(gpu, dtype, n, C, K):
    z, values, ids, rest, w = inputs(n, C, K, dtype, n + C)
    check(z, values, ids)
    check(z, values, ids, rest, 2.0, w)
    check(z, values, ids, None, 3.0, w, "sum")
    check(z, values, ids.long(), rest, 1.5, None, "none")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,C,K", [(600, 16, 3), (500, 17, 9), (600, 400, 4), (300, 255, 33), (300, 513, 16), (64, 700, 8),
                                   (64, 1024, 40), (60, 1025, 2), (30, 2500, 64), (40, 8200, 8), (300, 20_000, 4)])
def test_more_of_every_path(gpu, dtype, n, C, K):
    z, values, ids, rest, w = inputs(n, C, K, dtype, n + C, spread=6.0)
    check(z, values, ids, rest, 3.0, w)
    check(z, values, ids, None, 1.0, None, "none")


@pytest.mark.parametrize("value_type", TYPES)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_types_of_the_entries(gpu, value_type, reduction):
    z, values, ids, rest, w = inputs(90, 60, 6, torch.bfloat16, 1, torch.int64, value_type)
    check(z, values, ids, rest, 4.0, w, reduction)


def test_one_entry_is_cross_entropy(gpu):
    z, _, _, _, _ = inputs(500, 41, 1, torch.float32, 2)
    labels = torch.randint(0, 41, (500,), device="cuda")
    loss, dz = check(z, torch.zeros((500, 1), device="cuda"), labels.view(-1, 1))
    z64 = z.double().requires_grad_()
    want = torch.nn.functional.cross_entropy(z64, labels)
    want.backward()
    E = (41 / 64 + 300) * U  # check() has the closer bounds; of log q up to 10, and of q / 500
    assert abs(float(loss) - float(want.detach())) < 10 * E
    assert float((dz.double() - 0.75 * z64.grad).abs().max()) < 2 * E / 500


def test_a_student_that_is_the_teacher(gpu):
    """All entries and the rest: no loss, no gradient, but for roundings."""
    from tcc_amd import training

    z = torch.randn((200, 300), device="cuda") * 3
    entries = training.top_logits(z, 20, temperature=2.0)
    loss, dz = check(z, *entries, T=2.0)
    E = (300 / 64 + 300) * U  # of T^2 times the sum of p, and of T / n times p and q
    assert abs(float(loss)) < 4 * 4 * E and float(dz.abs().max()) < 2 * 2 * E / 200


@pytest.mark.parametrize("C,K", [(5, 12), (40, 8), (300, 64), (6000, 40)])
@pytest.mark.parametrize("rested", [False, True])
def test_the_same_class_in_several_entries(gpu, C, K, rested):
    gen = torch.Generator().manual_seed(C)
    n = 50
    z = torch.randn((n, C), generator=gen).cuda()
    ids = torch.randint(0, min(C, 6), (n, K), generator=gen) * (C // 6 if C > 6 else 1)
    ids[3] = ids[3, 0]
    values = torch.randn((n, K), generator=gen).cuda()
    rest = torch.randn(n, generator=gen).cuda() if rested else None
    check(z, values, ids.cuda(), rest, 2.0, None, "none")


@pytest.mark.parametrize("C", [9, 200, 6000])
def test_ids_outside_are_no_entries_and_reported(gpu, C):
    z, values, ids, rest, w = inputs(40, C, 5, torch.float32, 6)
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    version = error._version
    check(z, values, ids, rest, 1.0, w, "none", error)
    assert int(error) == 0 and error._version > version
    ids[4, 2], ids[7, 0], ids[9] = C, -2, 2**31 - 1
    check(z, values, ids, rest, 1.0, None, "none", error)
    assert int(error) == 7  # TCC_DEVERR_FEATURE_INDEX
    check(z, values, ids.long() + 2**33 * (ids < 0), None, 1.0, None, "none")


@pytest.mark.parametrize("C", [6, 90, 700, 6000])
@pytest.mark.parametrize("rested", [False, True])
def test_masked_classes_and_rows(gpu, C, rested):
    """Classes of -inf have no probability; what a row of weight 0 holds does not
    matter; a row whose entries are all -inf has no loss."""
    from tcc_amd import training

    z, values, ids, rest, w = inputs(60, C, 3, torch.float32, 7, some_absent=False)
    rest = rest if rested else None
    keep = torch.zeros_like(z, dtype=torch.bool).scatter_(1, ids.long(), True)
    keep.scatter_(1, keep.int().argmin(1, keepdim=True), True)  # one of the others
    z[(torch.rand(z.shape, device="cuda") < 0.5) & ~keep] = -np.inf
    values[5] = -np.inf
    w[:] = 1.0
    clean = check(z, values, ids, rest, 2.0, w, "none")
    w[10:20] = 0.0
    z[10], z[11], z[12] = np.nan, np.inf, -np.inf
    values[13], ids[14] = np.nan, 2**30
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    loss, stats, total = training.distill_loss(z, values, ids, rest=rest, temperature=2.0, weight=w, device_error=error)
    dz = training.distill_grad(torch.ones((), device="cuda"), z, values, ids, stats, rest=rest, temperature=2.0, weight=w,
                               total=total)
    assert int(error) == 0 and float(total) == 50.0 and bool(torch.isfinite(loss))
    assert bool((dz[10:20] == 0).all()) and bool((stats[10:20] == 0).all())
    rows = torch.cat([clean[0][:10], clean[0][20:]]).double()
    assert abs(float(loss) - float(rows.sum() / 50)) <= 4 * U * float(rows.sum() / 50)
    for p, q in ((dz[:10], clean[1][:10]), (dz[20:], clean[1][20:])):
        assert bool(((p * 50 * 0.75 - q).abs() <= 8 * U * q.abs() + 1e-12).all())


def test_what_has_no_finite_loss(gpu):
    """By the formula: infinite where the teacher has what the student rules out,
    NaN where a row of the student is NaN or nothing but -inf."""
    from tcc_amd import training

    z = torch.zeros((5, 10), device="cuda")
    ids = torch.tensor([[1, 2]] * 5, device="cuda")
    values = torch.zeros((5, 2), device="cuda")
    z[0, 1] = -np.inf
    z[1, 5] = np.nan
    z[2] = -np.inf
    values[3, 0] = np.nan
    loss, stats, _ = training.distill_loss(z, values, ids, reduction="none")
    assert float(loss[0]) == np.inf and bool(loss[1:4].isnan().all()) and bool(torch.isfinite(loss[4]))
    dz = training.distill_grad(torch.ones(5, device="cuda"), z, values, ids, stats, reduction="none")
    assert float(dz[0, 1]) == -0.5 and bool(torch.isfinite(dz[0]).all()) and bool(torch.isfinite(dz[4]).all())
    # a teacher that leaves something, a student that leaves nothing
    z[0] = -np.inf
    z[0, 1:3] = 0.0
    loss, stats, _ = training.distill_loss(z, values, ids, rest=torch.zeros(5, device="cuda"), reduction="none")
    assert float(loss[0]) == np.inf


def test_weights_that_add_to_nothing(gpu):
    z, values, ids, rest, w = inputs(30, 50, 4, torch.float32, 8)
    w.zero_()
    loss, dz = check(z, values, ids, rest, 1.0, w)
    assert float(loss) == 0.0 and bool((dz == 0).all())


def test_no_rows(gpu):
    from tcc_amd import training

    z, values = torch.empty((0, 9), device="cuda"), torch.empty((0, 4), device="cuda")
    ids = torch.empty((0, 4), dtype=torch.int32, device="cuda")
    for reduction in ("mean", "sum", "none"):
        loss, stats, _ = training.distill_loss(z, values, ids, reduction=reduction)
        assert stats.shape == (0, 4) and bool((loss == 0).all())
        assert training.distill_grad(torch.ones_like(loss), z, values, ids, stats, reduction=reduction).shape == (0, 9)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignments(gpu, dtype):
    """The same bits as dense copies'."""
    from tcc_amd import training

    z, values, ids, rest, w = inputs(40, 6000, 12, dtype, 9, some_absent=False)
    ids = ids % 40
    both = torch.stack([rest, w], 1)
    for cols in (slice(1, 48), slice(3, 503), slice(5, 5998)):
        a = z[:, cols], values[:, 1:8], ids[:, 1:8]
        check(*a, both[:, 0], 2.0, both[:, 1])
        dense = [t.contiguous() for t in a]
        for p, q in zip(training.distill_loss(*a, rest=both[:, 0]), training.distill_loss(*dense, rest=rest)):
            assert p is q is None or torch.equal(p, q)
    turned = z[:, :99].t().contiguous().t()
    check(turned, values, ids)


def test_large_logits_lose_nothing(gpu):
    """Levels far from zero leave the differences' digits."""
    z, values, ids, rest, w = inputs(60, 200, 6, torch.float32, 10, some_absent=False)
    check(z + 4096.0, values - 4096.0, ids, rest - 4096.0, 2.0, w)
    check(z * 30, values * 30, ids, rest, 2.0, w)


@pytest.mark.parametrize("T", [1e-18, 1e-4, 1e4, 1e15])
@pytest.mark.parametrize("C", [9, 150, 700, 6000])
def test_extreme_temperatures(gpu, C, T):
    z, values, ids, rest, w = inputs(50, C, 4, torch.float32, C)
    T = float(np.float32(T))
    check(z, values, ids, rest, T, w)
    check(z, values, ids, None, T, w, "none")


def test_many_rows(gpu):
    z, values, ids, rest, w = inputs(100_003, 20, 3, torch.float32, 11)
    check(z, values, ids, rest, 2.0, w)
    check(z, values, ids, None, 2.0, None)


@pytest.mark.parametrize("rested", [False, True])
def test_gradient_against_differences(gpu, rested):
    """Central differences of the 64-bit loss: off by the square of the step
    times third derivatives (below 1) and by 2^-53 over the step, 1e-8; the
    gradient's own bound is added."""
    from tcc_amd import training

    z, values, ids, rest, w = inputs(4, 9, 3, torch.float32, 12)
    rest = rest if rested else None
    loss, stats, total = training.distill_loss(z, values, ids, rest=rest, temperature=2.0, weight=w)
    dz = training.distill_grad(torch.ones((), device="cuda"), z, values, ids, stats, rest=rest, temperature=2.0, weight=w,
                               total=total).cpu()
    gtol = exact(z, values, ids, rest, 2.0, w, "mean")[3].view(-1)
    z64, s = z.double().cpu(), 1e-4
    for i in range(z.numel()):
        ends = []
        for sign in (1, -1):
            moved = z64.clone()
            moved.view(-1)[i] += sign * s
            ends.append(float(exact(moved, values, ids, rest, 2.0, w, "mean")[0]))
        assert abs((ends[0] - ends[1]) / (2 * s) - float(dz.view(-1)[i])) < 1e-7 + 2 * float(gtol[i])


def test_places_past_32_bits(gpu):
    """4.5e9 logits: the last rows'."""
    from tcc_amd import training

    n, C, K = 90_000, 50_000, 8
    z = torch.empty((n, C), dtype=torch.bfloat16, device="cuda").normal_()
    gen = torch.Generator().manual_seed(13)
    ids = torch.randint(0, C, (n, K), generator=gen, dtype=torch.int32).cuda()
    values = torch.randn((n, K), generator=gen).cuda()
    rest = torch.randn(n, generator=gen).cuda()
    loss, stats, _ = training.distill_loss(z, values, ids, rest=rest, reduction="none")
    dz = training.distill_grad(torch.ones(n, device="cuda"), z, values, ids, stats, rest=rest, reduction="none")
    end = slice(n - 20, n)
    rows, tol, grad, gtol = exact(z[end], values[end], ids[end], rest[end], 1.0, None, "none")
    assert bool(((loss[end].double().cpu() - rows).abs() <= tol).all())
    assert bool(((dz[end].double().cpu() - grad).abs() <= gtol + 2.0**-8 * (grad.abs() + gtol) + 1e-30).all())


def test_rows_of_two_billion_classes(gpu):
    """The longest rows: classes of which none but 70 count, at both ends and on
    the way, so that every sum is that of 70."""
    from tcc_amd import training

    C = 2**31 - 9
    places = torch.cat([torch.arange(20), C // 2 + torch.arange(25), C - 25 + torch.arange(25)]).cuda()
    near = torch.linspace(-4.0, 4.0, 70).roll(33).to(torch.bfloat16)[None].cuda()
    z = torch.full((1, C), -200.0, dtype=torch.bfloat16, device="cuda")
    z[:, places] = near
    values, ids, rest = training.top_logits(z, 8)
    want = torch.sort(near, dim=1, descending=True, stable=True)
    assert torch.equal(values, want.values[:, :8]) and torch.equal(ids[0].long(), places[want.indices[0, :8]])
    v, i, r = training.top_logits(near, 8)
    assert float((rest - r).abs()) <= 400 * U * (1 + float(r.abs()))
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    one = torch.ones((), device="cuda")
    for use in (None, rest):
        results = []
        for logits, at in ((z, ids), (near, i)):
            teacher = 0.5 * values
            loss, stats, _ = training.distill_loss(logits, teacher, at, rest=use, device_error=error)
            results.append((loss, training.distill_grad(one, logits, teacher, at, stats, rest=use)))
        (loss, dz), (loss_near, dz_near) = results
        assert float((loss - loss_near).abs()) <= 400 * U * (1 + float(loss_near.abs()))
        step = dz_near.float().abs() * 2 * U_OUT[torch.bfloat16] + 800 * U  # two roundings that may differ
        assert bool(((dz[:, places].float() - dz_near.float()).abs() <= step).all())
        dz[:, places] = 0
        assert float(dz.amax()) < 1e-30 and float(dz.amin()) >= 0
    assert int(error) == 0


def test_replayed_graph_and_other_stream(gpu):
    from tcc_amd import training

    gen = torch.Generator().manual_seed(4)
    for C in (90, 7000):
        z, values, ids, rest, w = inputs(500, C, 10, torch.float32, 14)
        one = torch.ones((), device="cuda")

        def both(stream=None):
            loss, stats, total = training.distill_loss(z, values, ids, rest=rest, temperature=2.0, weight=w, stream=stream)
            return loss, stats, training.distill_grad(one, z, values, ids, stats, rest=rest, temperature=2.0, weight=w,
                                                      total=total, stream=stream)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = both(side)
        torch.cuda.current_stream().wait_stream(side)
        for p, q in zip(got, both()):
            assert torch.equal(p, q)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both()
        for _ in range(3):
            z.copy_(torch.randn(z.shape, generator=gen))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for p, q in zip(out, both()):
                assert torch.equal(p, q)


def test_refusals_on_the_device(gpu):
    from tcc_amd import training

    z, v = torch.zeros((4, 10), device="cuda"), torch.zeros((4, 3), device="cuda")
    i = torch.zeros((4, 3), dtype=torch.int32, device="cuda")
    loss, stats, total = training.distill_loss(z, v, i, weight=z[:, 0])
    one = torch.ones((), device="cuda")
    for bad in (lambda: training.distill_loss(z, v[:3], i), lambda: training.distill_loss(z, v, i[:, :2]),
                lambda: training.distill_loss(z[0], v, i), lambda: training.distill_loss(z, v, i, rest=z[0]),
                lambda: training.distill_loss(z, v, i, weight=z[:3, 0]), lambda: training.distill_loss(z, v, i, temperature=-1.0),
                lambda: training.distill_loss(z, v, i, temperature=float("inf")),
                lambda: training.distill_loss(z, v, i, reduction="most"),
                lambda: training.distill_loss(z, v[:, :0], i[:, :0]),
                lambda: training.distill_loss(z, v[:, :1].expand(4, 65), i[:, :1].expand(4, 65)),
                lambda: training.distill_grad(one, z, v, i, stats[:3]), lambda: training.distill_grad(z[0], z, v, i, stats),
                lambda: training.distill_grad(one, z, v, i, stats, reduction="none"),
                lambda: training.distill_grad(one, z, v, i, stats, weight=z[:, 0])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: training.distill_loss(z.double(), v, i), lambda: training.distill_loss(z, v, i.short()),
                lambda: training.distill_loss(z, v, i, rest=z[:, 0].half()), lambda: training.distill_loss(z, v, i, weight=z[:, 0].cpu()),
                lambda: training.distill_grad(one.double(), z, v, i, stats)):
        with pytest.raises(TypeError):
            bad()
