"""Group norm over the rows of each graph with its activation, and its
gradient (tcc_amd.training), against plain 64-bit evaluations.

Bounds, with u = 2^-24 and K = 64 u: sums over these sizes run at most about
40 additions deep (rows of a lane, the lanes, the tiles), so a mean is off by
at most K max|x| and a standard deviation by K of itself and of that; z is
then off by K (|w| (|xh| + max|x| rstd) + |b|), and every activation has a
slope below 1.2 (its own functions are good to a few u of z).  One rounding
to the output's type is added.  The gradient takes the forward's mean and
rstd as given, and its mask from z in the rounding that both passes use."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

K = 64 * 2.0**-24
U_OUT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "silu", "gelu"]


def act64(name, z):
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    p = torch.special.ndtr(z)
    return z * p, p + z * torch.exp(-z * z / 2) / np.sqrt(2 * np.pi)


def forward64(x, G, w, b, at, eps, act):
    """(y, tolerance, mean, rstd) on the CPU, segment by segment."""
    N, C = x.shape
    x = x.double().cpu()
    w = torch.ones(C, dtype=torch.float64) if w is None else w.double().cpu()
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.double().cpu()
    y, tol = torch.zeros_like(x), torch.zeros_like(x)
    mean, rstd = torch.zeros(len(at) - 1, G).double(), torch.full((len(at) - 1, G), eps**-0.5).double()
    top = torch.zeros_like(mean)
    for i, (lo, hi) in enumerate(zip(at[:-1], at[1:])):
        if lo == hi:
            continue
        v = x[lo:hi].view(hi - lo, G, C // G)
        mean[i] = v.mean((0, 2))
        rstd[i] = (v.var((0, 2), unbiased=False) + eps) ** -0.5
        top[i] = v.abs().amax((0, 2))
        xh = (v - mean[i].view(1, G, 1)) * rstd[i].view(1, G, 1)
        z = (xh.reshape(hi - lo, C)) * w + b
        y[lo:hi] = act64(act, z)[0]
        reach = (xh.abs() + (top[i] * rstd[i]).view(1, G, 1)).reshape(hi - lo, C)
        tol[lo:hi] = 1.2 * K * (w.abs() * reach + b.abs())
    return y, tol, mean, rstd, top


def segments(kind, N, gen):
    if kind == "one":
        return None, [0, N]
    if kind == "ragged":  # with empty segments, at the ends too, and segments of one row
        cuts = torch.randint(0, N + 1, (max(1, N // 9),), generator=gen)
        at = torch.sort(torch.cat([torch.tensor([0, 0, N, N, min(1, N)]), cuts])).values
    else:  # two: a short and a long one
        at = torch.tensor([0, min(3, N), N])
    return at, at.tolist()


CASES = [(1, 1, 1), (1, 8, 2), (2, 6, 3), (37, 64, 8), (300, 100, 4), (1000, 256, 32), (513, 33, 11), (129, 602, 14),
         (700, 24, 1), (50, 2048, 16), (66, 1030, 2), (4000, 16, 16)]


def inputs(N, C, dtype, seed, offset=1.5):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn((N, C), generator=gen) * (torch.rand(C, generator=gen) + 0.3) + offset).to(dtype).cuda()
    w = (torch.rand(C, generator=gen) + 0.5).cuda()
    b = torch.randn(C, generator=gen).cuda()
    d = torch.randn((N, C), generator=gen).to(dtype).cuda()
    return gen, x, w, b, d


def check_forward(got, x, G, w, b, at, eps, act):
    y, mean, rstd = got
    y64, tol, m64, r64, top = forward64(x, G, w, b, at, eps, act)
    assert bool(((mean.double().cpu() - m64).abs() <= K * top + 1e-30).all())
    assert bool(((rstd.double().cpu() - r64).abs() <= K * r64 * (1 + top * r64)).all())
    tol = tol + U_OUT[y.dtype] * (y64.abs() + tol) + (2.0**-25 if y.dtype == torch.float16 else 0.0)
    err = (y.double().cpu() - y64).abs()
    assert bool((err <= tol).all()), f"largest excess {float((err - tol).max()):.3e}"


def check_grad(got, d, x, mean, rstd, G, w, b, at, act):
    dx, dw, db = got
    N, C = x.shape
    size = C // G
    w32 = torch.ones(C) if w is None else w.float().cpu()
    b32 = torch.zeros(C) if b is None else b.float().cpu()
    x32, mean, rstd = x.float().cpu(), mean.cpu(), rstd.cpu()
    dx64, tol = torch.zeros((N, C)).double(), torch.zeros((N, C)).double()
    sums = torch.zeros((4, C)).double()
    for i, (lo, hi) in enumerate(zip(at[:-1], at[1:])):
        if lo == hi:
            continue
        spread = lambda s: s[i].view(G, 1).expand(G, size).reshape(C)  # noqa: E731
        xh32 = (x32[lo:hi] - spread(mean)) * spread(rstd)
        z32 = xh32 * w32 + b32  # rounded after each operation, as the kernels do
        xh = (x32[lo:hi].double() - spread(mean).double()) * spread(rstd).double()
        z = xh * w32.double() + b32.double()
        slope = (z32 > 0).double() if act == "relu" else act64(act, z)[1]
        dy = d[lo:hi].double().cpu()
        dz, wd = dy * slope, w32.double()
        dxh = dz * wd
        over = lambda v: v.view(hi - lo, G, size).mean((0, 2)).view(G, 1).expand(G, size).reshape(C)  # noqa: E731
        r = spread(rstd).double()
        dx64[lo:hi] = (dxh - over(dxh) - xh * over(dxh * xh)) * r
        # dz: 8 u of itself and what z's few u change of the slope (its own slope is below 1)
        e = dy.abs() * (8 * 2.0**-24 * (1 + (xh * wd).abs() + b32.double().abs()))
        near = e * wd.abs() + K * (over(dxh.abs()) + xh.abs() * over((dxh * xh).abs()))
        near = near + over(e * wd.abs()) + xh.abs() * over(e * wd.abs() * (xh.abs() + 1))
        tol[lo:hi] = near * r
        sums += torch.stack([dz.sum(0), (dz * xh).sum(0), (dz.abs() * K + e).sum(0),
                             ((dz * xh).abs() * K + e * (xh.abs() + 1)).sum(0)])
    tol = tol + U_OUT[dx.dtype] * (dx64.abs() + tol) + (2.0**-25 if dx.dtype == torch.float16 else 0.0)
    err = (dx.double().cpu() - dx64).abs()
    assert bool((err <= tol + 1e-30).all()), f"dx: largest excess {float((err - tol).max()):.3e}"
    for name, v, want, t in (("dbias", db, sums[0], sums[2]), ("dweight", dw, sums[1], sums[3])):
        if v is not None:
            err = (v.double().cpu() - want).abs()
            assert bool((err <= t + 1e-30).all()), f"{name}: largest excess {float((err - t).max()):.3e}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["one", "ragged", "two"])
@pytest.mark.parametrize("N,C,G", CASES)
def test_both_passes(gpu, dtype, kind, N, C, G):
    from tcc_amd import training

    gen, x, w, b, d = inputs(N, C, dtype, N + C)
    off, at = segments(kind, N, gen)
    off = None if off is None else off.to(torch.int32 if N % 2 else torch.int64).cuda()
    for k, act in enumerate(ACTS):
        longest = max(hi - lo for lo, hi in zip(at[:-1], at[1:]))
        for rows in ((None, longest) if kind != "one" else (None,)):
            got = training.group_norm(x, G, w, b, offsets=off, activation=act, max_rows=rows)
            check_forward(got, x, G, w, b, at, 1e-5, act)
            back = training.group_norm_grad(d, x, got[1], got[2], G, w, b, offsets=off, activation=act, max_rows=rows)
            check_grad(back, d, x, got[1], got[2], G, w, b, at, act)
            for p, q in zip(back, training.group_norm_grad(d, x, got[1], got[2], G, w, b, offsets=off, activation=act,
                                                           max_rows=rows)):
                assert torch.equal(p, q), "the same inputs give the same bits"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("long", [0, 9000])
@pytest.mark.parametrize("N,C,G,mean_rows", [(30_000, 64, 8, 15), (30_000, 24, 2, 20), (40_000, 33, 11, 150),
                                             (12_000, 520, 1, 7), (12_000, 606, 2, 100),
                                             (30_000, 48, 16, 15), (25_000, 308, 4, 120), (31_000, 36, 4, 9)])
def test_many_short_segments_with_a_long_one(gpu, dtype, long, N, C, G, mean_rows):
    """Over a thousand segments (a wave each) or hundreds (a workgroup each),
    with empty ones, and one that is too long for either, whether the
    longest is known or not."""
    from tcc_amd import training

    gen, x, w, b, d = inputs(N, C, dtype, N + C)
    cuts = torch.randint(0, N - long, ((N - long) // mean_rows,), generator=gen)
    at = torch.sort(torch.cat([torch.tensor([0, N - long, N]), cuts])).values
    off, at = at.cuda(), at.tolist()
    act = ["relu", "silu", "gelu"][TYPES.index(dtype)]
    first = None
    for rows in (None, max(hi - lo for lo, hi in zip(at[:-1], at[1:]))):
        got = training.group_norm(x, G, w, b, offsets=off, activation=act, max_rows=rows)
        back = training.group_norm_grad(d, x, got[1], got[2], G, w, b, offsets=off, activation=act, max_rows=rows)
        if first is None:
            first = got, back
            check_forward(got, x, G, w, b, at, 1e-5, act)
            check_grad(back, d, x, got[1], got[2], G, w, b, at, act)
        else:  # another split at most: the same values
            for p, q in zip(got + back, first[0] + first[1]):
                assert bool(torch.isfinite(p).all())
                assert float((p.double() - q.double()).norm() / q.double().norm()) <= (1e-6 if p.dtype == torch.float32 else 1e-3)


@pytest.mark.parametrize("weight,bias,ptype", [(False, False, torch.float32), (True, False, torch.float32),
                                               (False, True, torch.bfloat16), (True, True, torch.bfloat16),
                                               (True, True, torch.float16)])
def test_weight_and_bias_forms(gpu, weight, bias, ptype):
    from tcc_amd import training

    gen, x, w, b, d = inputs(210, 48, torch.bfloat16, 3)
    off, at = segments("ragged", 210, gen)
    w, b, off = (w.to(ptype) if weight else None), (b.to(ptype) if bias else None), off.cuda()
    got = training.group_norm(x, 6, w, b, offsets=off, activation="silu")
    check_forward(got, x, 6, w, b, at, 1e-5, "silu")
    back = training.group_norm_grad(d, x, got[1], got[2], 6, w, b, offsets=off, activation="silu")
    assert (back[1] is None) == (not weight) and (back[2] is None) == (not bias)
    check_grad(back, d, x, got[1], got[2], 6, w, b, at, "silu")


def test_segments_of_one_size(gpu):
    """[B x ... x C]: what torch's group norm gives for channels first."""
    from tcc_amd import training

    gen, x, w, b, d = inputs(6 * 5 * 7, 40, torch.float32, 8)
    for shape in ((6, 35, 40), (6, 5, 7, 40), (210, 1, 40), (1, 210, 40)):
        B = shape[0]
        at = list(range(0, 211, 210 // B))
        v = x.view(shape)
        got = training.group_norm(v, 5, w, b, activation="relu")
        assert got[0].shape == v.shape and got[1].shape == (B, 5)
        check_forward((got[0].view(210, 40), *got[1:]), x, 5, w, b, at, 1e-5, "relu")
        back = training.group_norm_grad(d.view(shape), v, got[1], got[2], 5, w, b, activation="relu")
        check_grad((back[0].view(210, 40), *back[1:]), d, x, got[1], got[2], 5, w, b, at, "relu")
    first = torch.randn((4, 40, 9), device="cuda")  # channels first: copied
    got = training.group_norm(first.transpose(1, 2), 5)[0].transpose(1, 2)
    want = torch.nn.functional.group_norm(first.double().cpu(), 5)
    assert bool(((got.double().cpu() - want).abs() <= K * (want.abs() + 8)).all())


def test_strided_rows_are_read_in_place(gpu):
    from tcc_amd import training

    gen, x, w, b, d = inputs(300, 96, torch.float32, 5)
    off, at = segments("ragged", 300, gen)
    off = off.cuda()
    for cols in (slice(0, 32), slice(4, 36), slice(1, 31)):  # 16-byte and odd starts
        C = cols.stop - cols.start
        v, e = x[:, cols], d[:, cols]
        got = training.group_norm(v, 2, w[cols], b[cols], offsets=off)
        check_forward(got, v, 2, w[cols], b[cols], at, 1e-5, "none")
        back = training.group_norm_grad(e, v, got[1], got[2], 2, w[cols], b[cols], offsets=off)
        check_grad(back, e, v, got[1], got[2], 2, w[cols], b[cols], at, "none")
    one = d[:1].expand(300, 96)  # a broadcast gradient
    got = training.group_norm(x, 3, w, b, offsets=off)
    check_grad(training.group_norm_grad(one, x, got[1], got[2], 3, w, b, offsets=off), one, x, got[1], got[2], 3, w, b,
               at, "none")


@pytest.mark.parametrize("dtype,level", [(torch.float32, 3000.0), (torch.float32, -1e6), (torch.float16, 500.0)])
def test_large_means_lose_nothing(gpu, dtype, level):
    """Values far from zero against their spread: the variance comes from
    deviations, not from a difference of large sums."""
    from tcc_amd import training

    gen, x, w, b, _ = inputs(5000, 32, dtype, 13, offset=level)
    got = training.group_norm(x, 4, w, b)
    v = x.double().cpu().view(5000, 4, 8)
    mean, var = v.mean((0, 2)), v.var((0, 2), unbiased=False)
    assert bool(((got[1].double().cpu()[0] - mean).abs() <= K * mean.abs()).all())
    # deviations are taken from means that are off by K |mean| at most
    off = 2 * K * mean.abs() * var.sqrt() + (K * mean.abs()) ** 2 + K * var
    assert bool(((got[2].double().cpu()[0] ** -2 - 1e-5 - var).abs() <= 2 * off + 1e-9).all())


@pytest.mark.parametrize("size", [100.0, 1e4, 1e6])
@pytest.mark.parametrize("N,C,G,B", [(40_000, 64, 8, 1), (20_000, 30, 10, 1), (3000, 64, 8, 10), (3500, 12, 4, 2),
                                     (510, 100, 4, 3), (510, 150, 6, 600), (20, 64, 4, 1500), (300, 33, 11, 40)])
def test_outliers_among_the_first_rows(gpu, N, C, G, B, size):
    """Rows of many standard deviations where the kernels take what deviations
    are measured from: the first rows, and those at the quarters.  A lane adds
    some hundred deviations, whose roundings come as independent ones to 8 u of
    the sum and of the squares; joins add a few u more.  32 u for the standard
    deviation, and for the mean in units of it."""
    from tcc_amd import training

    gen = torch.Generator().manual_seed(17)
    for rows in ([0], [0, N // 4, N // 2, 3 * N // 4], list(range(min(N // 2, 40)))):
        x = torch.randn((B, N, C), generator=gen) + 0.5
        x[:, rows] *= size
        got = training.group_norm(x.cuda(), G)
        v = x.double().view(B, N, G, C // G)
        mean, var = v.mean((1, 3)), v.var((1, 3), unbiased=False)
        assert bool(((got[1].double().cpu() - mean).abs() <= 32 * 2.0**-24 * (var.sqrt() + mean.abs())).all())
        assert bool((got[2].double().cpu() * (var + 1e-5).sqrt() - 1).abs().max() <= 32 * 2.0**-24)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G", [1, 16, 4096])
@pytest.mark.parametrize("first", [0, 1])
def test_the_most_channels(gpu, dtype, G, first):
    """4,096 channels, in rows that begin aligned and in rows that do not."""
    from tcc_amd import training

    gen, x, w, b, d = inputs(70, 4104, dtype, G + first)
    cols = slice(first, first + 4096)
    x, w, b, d = x[:, cols], w[cols], b[cols], d[:, cols]
    for kind in ("one", "ragged"):
        off, at = segments(kind, 70, gen)
        off = None if off is None else off.cuda()
        got = training.group_norm(x, G, w, b, offsets=off, activation="silu")
        check_forward(got, x, G, w, b, at, 1e-5, "silu")
        back = training.group_norm_grad(d, x, got[1], got[2], G, w, b, offsets=off, activation="silu")
        check_grad(back, d, x, got[1], got[2], G, w, b, at, "silu")


@pytest.mark.parametrize("tail", [300, 200_000])
def test_places_past_32_bits(gpu, tail):
    """4.5e9 elements: the last segment's, whole and by tiles."""
    from tcc_amd import training

    N, C, G = 1_100_000, 4096, 8
    x, d = (torch.empty((N, C), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    x.normal_()
    d.normal_()
    x[N - tail:] += 2
    cuts = [0, N - tail, N] if tail > 1000 else list(range(0, N - tail, 1000)) + [N - tail, N]
    off = torch.tensor(cuts, device="cuda")
    y, mean, rstd = training.group_norm(x, G, offsets=off, activation="relu", max_rows=max(np.diff(cuts)).item())
    dx = training.group_norm_grad(d, x, mean, rstd, G, offsets=off, activation="relu", max_rows=max(np.diff(cuts)).item())[0]
    v, xt = x[N - tail:].view(tail, G, C // G), x[N - tail:]
    m64 = torch.stack([v[:, g].double().mean() for g in range(G)])
    s64 = torch.stack([v[:, g].double().var(unbiased=False) for g in range(G)])
    assert bool(((mean[-1].double() - m64).abs() <= K * 8).all())
    assert bool((rstd[-1].double() * (s64 + 1e-5).sqrt() - 1).abs().max() <= K * 8)
    m, r = (t[-1].view(G, 1).expand(G, C // G).reshape(C) for t in (mean, rstd))
    xh = (xt[-200:].float() - m) * r
    want = xh.clamp(min=0).to(torch.bfloat16)
    assert torch.equal(y[-200:], want)
    dz = torch.where((v.float() - mean[-1].view(1, G, 1)) * rstd[-1].view(1, G, 1) > 0, d[N - tail:].view(v.shape).float(), 0.0)
    xv = (v.float() - mean[-1].view(1, G, 1)) * rstd[-1].view(1, G, 1)
    s1 = dz.double().mean((0, 2)).view(G, 1).expand(G, C // G).reshape(C)
    s2 = torch.stack([(dz[:, g].double() * xv[:, g].double()).mean() for g in range(G)]).view(G, 1).expand(G, C // G).reshape(C)
    want = (dz[-200:].reshape(200, C).double() - s1 - xh.double() * s2) * r.double()
    tol = 2.0**-8 * want.abs() + K * (s1.abs() + s2.abs() * xh.abs() + dz[-200:].reshape(200, C).abs() + 1) * r.double()
    assert bool(((dx[-200:].double() - want).abs() <= tol).all())


def test_constant_and_non_finite_groups(gpu):
    from tcc_amd import training

    x = torch.full((40, 8), 7.0, device="cuda")
    y, mean, rstd = training.group_norm(x, 2)
    assert bool((y == 0).all()) and bool((mean == 7).all())
    x[25, 1] = float("inf")
    off = torch.tensor([0, 20, 20, 40], device="cuda")
    y, mean, rstd = training.group_norm(x, 2, offsets=off, activation="relu")
    assert bool(torch.isfinite(y[:20]).all()) and bool(torch.isfinite(y[:, 4:]).all())
    assert bool(y[20:, :4].isnan().all()), "a group that holds an infinity has no mean"
    assert torch.equal(mean[1], torch.zeros(2, device="cuda"))


def test_no_rows(gpu):
    from tcc_amd import training

    x = torch.empty((0, 12), device="cuda")
    w = torch.ones(12, device="cuda")
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    y, mean, rstd = training.group_norm(x, 3, w, w, offsets=off)
    assert y.shape == (0, 12) and mean.shape == (3, 3) and bool((mean == 0).all())
    dx, dw, db = training.group_norm_grad(x, x, mean, rstd, 3, w, w, offsets=off)
    assert dx.shape == (0, 12) and bool((dw == 0).all()) and bool((db == 0).all())


@pytest.mark.parametrize("shape,G", [((0, 12), 3), ((1, 0, 12), 3), ((7, 0, 12), 12), ((1000, 0, 2, 24), 24), ((0, 5, 12), 3)])
def test_segments_of_one_size_without_rows(gpu, shape, G):
    """No offsets and no rows: every segment is empty, in number above what
    the workspace has room for beside slots."""
    from tcc_amd import training

    B = 1 if len(shape) == 2 else shape[0]
    x, w = torch.empty(shape, device="cuda"), torch.ones(shape[-1], device="cuda")
    y, mean, rstd = training.group_norm(x, G, w, w, eps=0.25)
    assert y.shape == shape and mean.shape == (B, G)
    assert bool((mean == 0).all()) and bool((rstd == 2.0).all())
    dx, dw, db = training.group_norm_grad(x, x, mean, rstd, G, w, w)
    assert dx.shape == shape and bool((dw == 0).all()) and bool((db == 0).all())


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_gradient_against_differences(gpu, act):
    """The change of sum(d * y) along e, for x, weight and bias: central
    differences at h have an error of about h^2 times third derivatives
    (below 30 here) and u |y| / h a term."""
    from tcc_amd import training

    gen, x, w, b, d = inputs(150, 24, torch.float32, 21, offset=0.2)
    off = torch.tensor([0, 40, 90, 150], device="cuda")
    e = [torch.randn(t.shape, generator=gen).cuda() for t in (x, w, b)]
    f = lambda h: (training.group_norm(x + h * e[0], 4, w + h * e[1], b + h * e[2], offsets=off,  # noqa: E731
                                       activation=act)[0].double() * d.double()).sum()
    y, mean, rstd = training.group_norm(x, 4, w, b, offsets=off, activation=act)
    back = training.group_norm_grad(d, x, mean, rstd, 4, w, b, offsets=off, activation=act)
    along = float(sum((p.double() * q.double()).sum() for p, q in zip(back, e)))
    h = 1e-2
    quotient = float((f(h) - f(-h)) / (2 * h))
    tol = 30 * h * h * d.numel() ** 0.5 + 16 * 2.0**-24 / h * float((d.abs() * (y.abs() + 1)).sum())
    assert abs(along - quotient) <= tol


def test_gradient_of_more_than_a_launch(gpu):
    """Rows of 129 vectors, two to a workgroup: more workgroups than one launch
    has threads for (69 GB each of x and dx).  x = dy = +-1 in turn with mean 0
    and rstd 1/2: dx = (x - 0 - x / 4) / 2, off by what the sums' fp32 is."""
    from tcc_amd import training

    N, C = 2**25 + 999, 516
    x = torch.ones((N, C), device="cuda")
    x[1::2] = -1
    mean, rstd = torch.zeros((1, 1), device="cuda"), torch.full((1, 1), 0.5, device="cuda")
    dx, _, _ = training.group_norm_grad(x, x, mean, rstd, 1)
    for at in range(0, N, 2**22):
        assert float((dx[at:at + 2**22] - 0.375 * x[at:at + 2**22]).abs().max()) < 1e-3


@pytest.mark.parametrize("spread", [0.3, 1.0, 4.0])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_fp32_activations_are_as_good_as_plain_ones(gpu, act, spread):
    """The activations and their slopes at the z that the kernels form: every
    operation of a plain evaluation in 32 bits rounds by at most u = 2^-24,
    0.4 u in the mean, and a handful of them leave a relative L2 error below u.
    One row whose dy is 1 gives the slopes as dBias."""
    from tcc_amd import training

    gen = torch.Generator().manual_seed(31)
    N, C = 64, 4096
    x = torch.randn((N, C), generator=gen).cuda()
    w = (torch.rand(C, generator=gen) * 0.5 + 0.75).mul_(spread).cuda()
    b = (torch.randn(C, generator=gen) * 0.3).cuda()
    rel = lambda a, v: float((a.double().cpu() - v).norm() / v.norm())  # noqa: E731
    y, mean, rstd = training.group_norm(x, 1, w, b, activation=act)
    z = ((x - mean) * rstd) * w + b  # rounded after each operation, as the kernels do
    assert rel(y, act64(act, z.double().cpu())[0]) <= 2.0**-24
    one = x[:1].contiguous()
    dy, zero, unit = torch.ones_like(one), torch.zeros_like(mean), torch.ones_like(rstd)
    _, _, db = training.group_norm_grad(dy, one, zero, unit, 1, w, b, activation=act)
    assert rel(db, act64(act, (one * w + b)[0].double().cpu())[1]) <= 2.0**-24
    far = torch.linspace(-60.0, 60.0, C, device="cuda").view(1, C)  # both tails, and none of them not finite
    dx, _, db = training.group_norm_grad(dy, far, zero.expand(1, C).contiguous(), unit.expand(1, C).contiguous(), C, w, b,
                                         activation=act)
    assert bool(torch.isfinite(dx).all()) and bool(torch.isfinite(db).all())
    slope = act64(act, (far * w + b)[0].double().cpu())[1]
    assert bool(((db.double().cpu() - slope).abs() <= 8 * 2.0**-24).all())


def test_relu_mask_is_the_forward_s(gpu):
    """Values that land on zero or beside it: dy passes exactly where y > 0."""
    from tcc_amd import training

    gen, x, w, _, _ = inputs(64, 16, torch.float32, 2)
    y0, mean, rstd = training.group_norm(x, 16, w)
    b = -y0[5].clone()  # row 5 lands on zero
    y, mean, rstd = training.group_norm(x, 16, w, b, activation="relu")
    assert bool((y[5] == 0).all())
    d = torch.zeros_like(x)
    d[5] = 1.0
    dx, dw, db = training.group_norm_grad(d, x, mean, rstd, 16, w, b, activation="relu")
    assert bool((db == 0).all()) and bool((dx == 0).all())


@pytest.mark.parametrize("maxRows, C, G", [(40, 32, 4), (None, 32, 4), (40, 30, 10), (5000, 32, 4)])
def test_relu_masks_infinities(gpu, maxRows, C, G):
    """An infinite dy where relu masks is as good as none, and a bias of -inf
    leaves zeros: in whole segments, in groups that vectors straddle, in tiles."""
    from tcc_amd import training

    each = maxRows or 40
    gen, x, w, b, d = inputs(5 * each, C, torch.float32, 12)
    off = None if maxRows else torch.arange(0, 5 * each + 1, each, device="cuda")
    if off is None:
        x, d = x.view(5, each, C), d.view(5, each, C)
    y, mean, rstd = training.group_norm(x, G, w, b, offsets=off, activation="relu")
    at = [each * i for i in range(6)]
    none = torch.where(y > 0, d, 0.0)
    flat = lambda t: t.reshape(5 * each, C)  # noqa: E731
    for masked in (float("inf"), -float("inf"), float("nan")):
        got = training.group_norm_grad(torch.where(y > 0, d, masked), x, mean, rstd, G, w, b, offsets=off,
                                       activation="relu")
        check_grad((flat(got[0]), *got[1:]), flat(none), flat(x), mean, rstd, G, w, b, at, "relu")
    b[3] = -float("inf")
    y2 = training.group_norm(x, G, w, b, offsets=off, activation="relu")[0]
    y[..., 3] = 0.0
    assert torch.equal(y2, y)


def test_replayed_graph_and_other_stream(gpu):
    from tcc_amd import training

    gen, x, w, b, d = inputs(3000, 64, torch.float32, 4)
    off, at = segments("ragged", 3000, gen)
    off = off.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = training.group_norm(x, 8, w, b, offsets=off, activation="gelu", stream=side)
    back = training.group_norm_grad(d, x, got[1], got[2], 8, w, b, offsets=off, activation="gelu", stream=side)
    torch.cuda.current_stream().wait_stream(side)
    check_forward(got, x, 8, w, b, at, 1e-5, "gelu")
    check_grad(back, d, x, got[1], got[2], 8, w, b, at, "gelu")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = training.group_norm(x, 8, w, b, offsets=off, activation="gelu")
        back = training.group_norm_grad(d, x, mean, rstd, 8, w, b, offsets=off, activation="gelu")
    for _ in range(3):
        x.copy_(torch.randn(x.shape, generator=gen))
        d.copy_(torch.randn(x.shape, generator=gen))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = training.group_norm(x, 8, w, b, offsets=off, activation="gelu")
        for p, q in zip((y, mean, rstd), want):
            assert torch.equal(p, q)
        for p, q in zip(back, training.group_norm_grad(d, x, want[1], want[2], 8, w, b, offsets=off, activation="gelu")):
            assert torch.equal(p, q)
