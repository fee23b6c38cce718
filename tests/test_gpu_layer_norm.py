"""Layer norm of rows with the residual sum before it and the activation after
it, and its gradient (tcc_amd.training), against plain 64-bit evaluations.

Bounds, with u = 2^-24 and K = 64 u: sums over up to 16,384 channels run at most
about 40 additions deep (16 of a lane, ten steps over the lanes, the difference
from the first mean), so a mean is off by at most K max|h| and a standard
deviation by K of itself and of that; z is then off by
K (|w| (|xh| + max|h| rstd) + |b|), and every activation has a slope below 1.2.
The sum h is one rounding of the exact sum: equal bits.  The gradient takes the
forward's mean and rstd as given, and its mask from z in the rounding that both
passes use; the sums over rows of dw and db add a lane's rows one after the
other (16 of 4,000 rows here), sixteen teams, and the workgroups in 64 bits.
One rounding to the output's type is added."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

K = 64 * 2.0**-24
U_OUT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 1e-30, torch.bfloat16: 1e-30, torch.float16: 2.0**-25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "silu", "gelu"]
SHAPES = [(1, 1), (1, 2), (3, 3), (2, 7), (5, 9), (37, 64), (300, 100), (513, 33), (4000, 16), (1000, 256), (70, 301),
          (129, 602), (66, 1030), (50, 2048), (40, 2050), (9, 4097), (5, 16384), (3, 16383)]


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


def inputs(N, C, dtype, seed, offset=1.5):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn((N, C), generator=gen) * (torch.rand(C, generator=gen) + 0.3) + offset).to(dtype).cuda()
    r, d, e = (torch.randn((N, C), generator=gen).to(dtype).cuda() for _ in range(3))
    w = (torch.rand(C, generator=gen) + 0.5).cuda()
    b = torch.randn(C, generator=gen).cuda()
    return gen, x, r, w, b, d, e


def params64(w, b, C):
    w = torch.ones(C, dtype=torch.float64) if w is None else w.double().cpu()
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.double().cpu()
    return w, b


def check_forward(got, x, residual, w, b, eps, act):
    y, h, mean, rstd = got
    C = x.shape[-1]
    if residual is not None:
        assert torch.equal(h, (x.float() + residual.float()).to(x.dtype))
    v = h.double().cpu()
    w, b = params64(w, b, C)
    m64, top = v.mean(-1, keepdim=True), v.abs().amax(-1, keepdim=True)
    r64 = (v.var(-1, keepdim=True, unbiased=False) + eps) ** -0.5
    assert mean.shape == rstd.shape == x.shape[:-1]
    assert bool(((mean.double().cpu().unsqueeze(-1) - m64).abs() <= K * top + 1e-30).all())
    assert bool(((rstd.double().cpu().unsqueeze(-1) - r64).abs() <= K * r64 * (1 + top * r64)).all())
    xh = (v - m64) * r64
    y64 = act64(act, xh * w + b)[0]
    tol = 1.2 * K * (w.abs() * (xh.abs() + top * r64) + b.abs())
    tol = tol + U_OUT[y.dtype] * (y64.abs() + tol) + TINY[y.dtype]
    err = (y.double().cpu() - y64).abs()
    assert bool((err <= tol).all()), f"largest excess {float((err - tol).max()):.3e}"


def check_grad(got, d, h, mean, rstd, w, b, act, add=None):
    dx, dw, db = got
    C = h.shape[-1]
    w64, b64 = params64(w, b, C)
    h32, m32, r32 = h.float().cpu(), mean.cpu().unsqueeze(-1), rstd.cpu().unsqueeze(-1)
    z32 = ((h32 - m32) * r32) * w64.float() + b64.float()  # rounded after each operation, as the kernels do
    r = r32.double()
    xh = (h32.double() - m32.double()) * r
    z = xh * w64 + b64
    dy = d.double().cpu()
    dz = dy * ((z32 > 0).double() if act == "relu" else act64(act, z)[1])
    dxh = dz * w64
    over = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    want = (dxh - over(dxh) - xh * over(dxh * xh)) * r
    # dz: 8 u of itself and what z's few u change of the slope (its own slope is below 1)
    e = dy.abs() * (8 * 2.0**-24 * (1 + (xh * w64).abs() + b64.abs()))
    near = e * w64.abs() + K * (dxh.abs() + over(dxh.abs()) + xh.abs() * over((dxh * xh).abs()))
    tol = (near + over(e * w64.abs()) + xh.abs() * over(e * w64.abs() * (xh.abs() + 1))) * r
    if add is not None:
        want = want + add.double().cpu()
        tol = tol + 2 * 2.0**-24 * want.abs()
    tol = tol + U_OUT[dx.dtype] * (want.abs() + tol) + TINY[dx.dtype]
    err = (dx.double().cpu() - want).abs()
    assert bool((err <= tol).all()), f"dx: largest excess {float((err - tol).max()):.3e}"
    flat = lambda t: t.reshape(-1, C).sum(0)  # noqa: E731
    for name, v, want, t in (("dbias", db, flat(dz), flat(dz.abs() * K + e)),
                             ("dweight", dw, flat(dz * xh), flat((dz * xh).abs() * K + e * (xh.abs() + 1)))):
        if v is not None:
            err = (v.double().cpu() - want).abs()
            assert bool((err <= t + 1e-30).all()), f"{name}: largest excess {float((err - t).max()):.3e}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,C", SHAPES)
def test_both_passes(gpu, dtype, N, C):
    from tcc_amd import training

    _, x, res, w, b, d, e = inputs(N, C, dtype, N + C)
    for act in ACTS:
        for residual, add in ((None, None), (res, e)):
            got = training.layer_norm(x, w, b, residual=residual, activation=act)
            assert residual is not None or got[1] is x
            check_forward(got, x, residual, w, b, 1e-5, act)
            back = lambda: training.layer_norm_grad(d, got[1], got[2], got[3], w, b, d_sum=add, activation=act)  # noqa: E731
            first = back()
            check_grad(first, d, got[1], got[2], got[3], w, b, act, add)
            for p, q in zip(first, back()):
                assert torch.equal(p, q), "the same inputs give the same bits"


@pytest.mark.parametrize("N,C", [(20_011, 40), (9000, 301), (2100, 4000), (600, 16000), (40_000, 6)])
def test_more_rows_than_teams(gpu, N, C):
    from tcc_amd import training

    _, x, res, w, b, d, e = inputs(N, C, torch.float32, 5)
    got = training.layer_norm(x, w, b, residual=res, activation="relu")
    check_forward(got, x, res, w, b, 1e-5, "relu")
    check_grad(training.layer_norm_grad(d, got[1], got[2], got[3], w, b, d_sum=e, activation="relu"), d, got[1], got[2],
               got[3], w, b, "relu", e)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_width_of_team(gpu, dtype):
    """The last channels that a team holds, and the first that the next one does."""
    from tcc_amd import training

    for C in (4, 5, 8, 12, 17, 31, 32, 36, 65, 95, 128, 129, 192, 193, 255, 257, 383, 385, 511, 513, 767, 769, 1023, 1024, 1025,
              2047, 2049, 4095, 4096, 8191, 8192, 8193, 16_000):
        _, x, res, w, b, d, e = inputs(23, C, dtype, C)
        got = training.layer_norm(x, w, b, residual=res, activation="gelu")
        check_forward(got, x, res, w, b, 1e-5, "gelu")
        check_grad(training.layer_norm_grad(d, *got[1:], w, b, d_sum=e, activation="gelu"), d, *got[1:], w, b, "gelu", e)


@pytest.mark.parametrize("N,C,dtype,run", [(30_000_000, 6, torch.float32, 144), (1_300_000, 250, torch.float32, 144),
                                           (2_000_001, 257, torch.bfloat16, 144), (200_000, 4000, torch.bfloat16, 288),
                                           (70_001, 8192, torch.float32, 288), (60_000, 16_384, torch.float16, 288)])
def test_parameter_sums_over_many_rows(gpu, N, C, dtype, run):
    """A team's rows in several runs, each summed in 32 bits: at most `run` rows
    one after the other, whose sum is off by run u of the terms' sizes, and six
    roundings of each term; all else is in 64 bits."""
    from tcc_amd import training

    gen = torch.Generator(device="cuda").manual_seed(N)
    draw = lambda: torch.empty((N, C), dtype=dtype, device="cuda").normal_(generator=gen)  # noqa: E731
    x, d = draw(), draw()
    w, b = torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
    _, _, mean, rstd = training.layer_norm(x, w, b)
    _, dw, db = training.layer_norm_grad(d, x, mean, rstd, w, b)
    sums = torch.zeros((4, C), dtype=torch.float64, device="cuda")
    step = 100_000_000 // C
    for i in range(0, N, step):
        at = slice(i, i + step)
        xh = (x[at].double() - mean[at].double()[:, None]) * rstd[at].double()[:, None]
        terms = d[at].double(), d[at].double() * xh
        sums += torch.stack([t.sum(0) for v in terms for t in (v, v.abs())])
    for got, want, size in ((db, sums[0], sums[1]), (dw, sums[2], sums[3])):
        assert bool(((got.double() - want).abs() <= (run + 6) * 2.0**-24 * size).all())


@pytest.mark.parametrize("weight,bias,ptype", [(False, False, torch.float32), (True, False, torch.float32),
                                               (False, True, torch.bfloat16), (True, True, torch.bfloat16),
                                               (True, True, torch.float16)])
def test_weight_and_bias_forms(gpu, weight, bias, ptype):
    from tcc_amd import training

    _, x, _, w, b, d, _ = inputs(70, 90, torch.bfloat16, 3)
    w, b = w.to(ptype) if weight else None, b.to(ptype) if bias else None
    if weight:  # at an address that only its elements are aligned to
        w = torch.cat([w[:1], w])[1:]
    got = training.layer_norm(x, w, b, eps=1e-3, activation="silu")
    check_forward(got, x, None, w, b, 1e-3, "silu")
    back = training.layer_norm_grad(d, x, got[2], got[3], w, b, activation="silu")
    check_grad(back, d, x, got[2], got[3], w, b, "silu")
    for v, there in zip(back[1:], (weight, bias)):
        assert (v is not None) == there and (v is None or v.dtype == torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
def test_shapes_strides_and_alignments(gpu, dtype):
    """Rows of any stride and address, the same bits as a dense copy's; other
    numbers of dimensions; broadcast and transposed inputs."""
    from tcc_amd import training

    _, x, res, w, b, d, e = inputs(60, 96, dtype, 9)
    for cols in (slice(0, 32), slice(4, 36), slice(1, 31), slice(3, 93), slice(95, 96)):
        args = x[:, cols], w[cols], b[cols]
        got = training.layer_norm(*args, residual=res[:, cols], activation="gelu")
        want = training.layer_norm(args[0].contiguous(), *args[1:], residual=res[:, cols].contiguous(), activation="gelu")
        for p, q in zip(got, want):
            assert torch.equal(p, q)
        back = training.layer_norm_grad(d[:, cols], got[1], got[2], got[3], *args[1:], d_sum=e[:, cols], activation="gelu")
        check_grad(back, d[:, cols], got[1], got[2], got[3], *args[1:], "gelu", e[:, cols])
    cube = x.view(3, 20, 96)
    got = training.layer_norm(cube, w, b, residual=res.view(3, 20, 96))
    check_forward(got, cube, res.view(3, 20, 96), w, b, 1e-5, "none")
    check_grad(training.layer_norm_grad(d.view(3, 20, 96), got[1], got[2], got[3], w, b), d.view(3, 20, 96), got[1], got[2],
               got[3], w, b, "none")
    one = training.layer_norm(x[0], w, b)  # a single row
    assert one[2].shape == () and torch.equal(one[0], training.layer_norm(x[:1], w, b)[0][0])
    turned = x.t().contiguous().t()
    assert torch.equal(training.layer_norm(turned, w, b)[0], training.layer_norm(x, w, b)[0])
    wide = d[:1].expand(60, 96)  # a broadcast gradient
    got = training.layer_norm(x, w, b)
    check_grad(training.layer_norm_grad(wide, x, got[2], got[3], w, b), wide, x, got[2], got[3], w, b, "none")


@pytest.mark.parametrize("dtype,level", [(torch.float32, 3000.0), (torch.float32, -1e6), (torch.float16, 500.0)])
@pytest.mark.parametrize("C", [50, 4096])
def test_large_means_lose_nothing(gpu, dtype, level, C):
    """The variance of rows far from zero: that of their differences, not that
    of their squares.  The second mean leaves one rounding of the mean."""
    from tcc_amd import training

    _, x, _, _, _, _, _ = inputs(40, C, dtype, 7, offset=level)
    _, _, mean, rstd = training.layer_norm(x)
    v = x.double().cpu()
    m64 = v.mean(-1)
    var = v.var(-1, unbiased=False)
    assert bool(((mean.double().cpu() - m64).abs() <= 2 * 2.0**-24 * m64.abs() + K * var.sqrt()).all())
    assert bool((rstd.double().cpu() * (var + 1e-5).sqrt() - 1).abs().max() <= K)


def test_constant_and_non_finite_rows(gpu):
    from tcc_amd import training

    x = torch.full((6, 40), 7.0, device="cuda")
    y, _, mean, rstd = training.layer_norm(x)
    assert bool((y == 0).all()) and bool((mean == 7).all()) and bool((rstd * 1e-5**0.5 - 1).abs().max() < K)
    x[1, 3], x[2, 39], x[3, 0] = float("inf"), float("nan"), -float("inf")
    x[4] = 3e30  # squares past fp32
    x[4, ::2] = -3e30
    for act in ("none", "relu"):
        y, _, mean, rstd = training.layer_norm(x, activation=act)
        assert bool(y[1:4].isnan().all()), "a row that holds an infinity or a NaN has no mean"
        assert bool((y[[0, 4, 5]] == 0).all()) and bool((rstd[4] == 0).all())
    dx, _, _ = training.layer_norm_grad(torch.ones_like(x), x, mean, rstd)
    assert bool(torch.isfinite(dx[[0, 4, 5]]).all())
    y = training.layer_norm(x[:1], eps=0.0)[0]
    assert bool(y.isnan().all()), "a constant row without eps is 0 / 0"


def test_no_rows(gpu):
    from tcc_amd import training

    w, b = torch.ones(12, device="cuda"), torch.zeros(12, device="cuda")
    for shape in ((0, 12), (3, 0, 12)):
        x = torch.empty(shape, device="cuda")
        y, h, mean, rstd = training.layer_norm(x, w, b, residual=x)
        assert y.shape == h.shape == shape and mean.shape == rstd.shape == shape[:-1]
        dx, dw, db = training.layer_norm_grad(x, x, mean, rstd, w, b, d_sum=x)
        assert dx.shape == shape and bool((dw == 0).all()) and bool((db == 0).all())


def test_relu_mask_is_the_forward_s(gpu):
    """Values that land on zero or beside it: dy passes exactly where y > 0; an
    infinite dy where relu masks is as good as none."""
    from tcc_amd import training

    _, x, _, w, b, d, _ = inputs(64, 48, torch.float32, 2)
    b0 = -training.layer_norm(x, w)[0][5].clone()  # row 5 lands on zero
    y, _, mean, rstd = training.layer_norm(x, w, b0, activation="relu")
    assert bool((y[5] == 0).all())
    one = torch.zeros_like(x)
    one[5] = 1.0
    for t in training.layer_norm_grad(one, x, mean, rstd, w, b0, activation="relu"):
        assert bool((t == 0).all())
    y, _, mean, rstd = training.layer_norm(x, w, b, activation="relu")
    want = training.layer_norm_grad(torch.where(y > 0, d, 0.0), x, mean, rstd, w, b, activation="relu")
    for masked in (float("inf"), float("nan")):
        got = training.layer_norm_grad(torch.where(y > 0, d, masked), x, mean, rstd, w, b, activation="relu")
        for p, q in zip(got, want):
            assert torch.equal(p, q)


@pytest.mark.parametrize("spread", [0.3, 1.0, 4.0])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_fp32_activations_are_as_good_as_plain_ones(gpu, act, spread):
    """At the z that the kernels form: every operation of a plain evaluation in
    32 bits rounds by at most u = 2^-24, 0.4 u in the mean, and a handful of
    them leave a relative L2 error below u."""
    from tcc_amd import training

    gen = torch.Generator().manual_seed(31)
    x = torch.randn((64, 4096), generator=gen).cuda()
    w = (torch.rand(4096, generator=gen) * 0.5 + 0.75).mul_(spread).cuda()
    b = (torch.randn(4096, generator=gen) * 0.3).cuda()
    y, _, mean, rstd = training.layer_norm(x, w, b, activation=act)
    z = ((x - mean[:, None]) * rstd[:, None]) * w + b
    want = act64(act, z.double().cpu())[0]
    assert float((y.double().cpu() - want).norm() / want.norm()) <= 2.0**-24


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_gradient_against_differences(gpu, act):
    """Central differences of the 64-bit forward of a row; the gradient in fp32
    has its own K, differences of step s are off by s^2 times third derivatives
    (below 10 here) and by 2^-53 / s."""
    from tcc_amd import training

    _, x, _, w, b, d, _ = inputs(3, 13, torch.float32, 8)
    _, _, mean, rstd = training.layer_norm(x, w, b, activation=act)
    dx, dw, db = (t.double().cpu() for t in training.layer_norm_grad(d, x, mean, rstd, w, b, activation=act))

    def loss(x, w, b):
        xh = (x - x.mean(-1, keepdim=True)) * (x.var(-1, keepdim=True, unbiased=False) + 1e-5) ** -0.5
        return (act64(act, xh * w + b)[0] * d.double().cpu()).sum()

    at = [t.double().cpu() for t in (x, w, b)]
    s = 1e-4
    for k, grad in enumerate((dx, dw, db)):
        for i in range(at[k].numel()):
            ends = []
            for sign in (1, -1):
                moved = [t.clone() for t in at]
                moved[k].view(-1)[i] += sign * s
                ends.append(loss(*moved))
            assert abs(float((ends[0] - ends[1]) / (2 * s) - grad.view(-1)[i])) < 1e-4


def test_places_past_32_bits(gpu):
    """4.4e9 elements: the last rows'."""
    from tcc_amd import training

    N, C = 1_100_000, 4000
    x, d = (torch.empty((N, C), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    x.normal_()
    d.normal_()
    y, h, mean, rstd = training.layer_norm(x, residual=d, activation="relu")
    dx = training.layer_norm_grad(d, h, mean, rstd, d_sum=x, activation="relu")[0]
    end = slice(N - 40, N)
    check_forward((y[end], h[end], mean[end], rstd[end]), x[end], d[end], None, None, 1e-5, "relu")
    check_grad((dx[end], None, None), d[end], h[end], mean[end], rstd[end], None, None, "relu", x[end])


def test_replayed_graph_and_other_stream(gpu):
    from tcc_amd import training

    gen, x, r, w, b, d, e = inputs(3000, 100, torch.float32, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = training.layer_norm(x, w, b, residual=r, activation="gelu", stream=side)
    back = training.layer_norm_grad(d, *got[1:], w, b, d_sum=e, activation="gelu", stream=side)
    torch.cuda.current_stream().wait_stream(side)
    check_forward(got, x, r, w, b, 1e-5, "gelu")
    check_grad(back, d, *got[1:], w, b, "gelu", e)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = training.layer_norm(x, w, b, residual=r, activation="gelu")
        back = training.layer_norm_grad(d, *out[1:], w, b, d_sum=e, activation="gelu")
    for _ in range(3):
        for t in (x, r, d):
            t.copy_(torch.randn(x.shape, generator=gen))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = training.layer_norm(x, w, b, residual=r, activation="gelu")
        for p, q in zip(out, want):
            assert torch.equal(p, q)
        for p, q in zip(back, training.layer_norm_grad(d, *want[1:], w, b, d_sum=e, activation="gelu")):
            assert torch.equal(p, q)


def test_refusals_on_the_device(gpu):
    from tcc_amd import training

    x, w = torch.zeros((4, 6), device="cuda"), torch.zeros(6, device="cuda")
    s = torch.zeros(4, device="cuda")
    for bad in (lambda: training.layer_norm(x, w[:5]), lambda: training.layer_norm(x, w, w.half()),
                lambda: training.layer_norm(x, residual=x.half()), lambda: training.layer_norm(x, residual=x[:3]),
                lambda: training.layer_norm(x, eps=-1.0), lambda: training.layer_norm(x, activation="tanh"),
                lambda: training.layer_norm(torch.zeros((2, 16385), device="cuda")),
                lambda: training.layer_norm(torch.zeros((2, 0), device="cuda")),
                lambda: training.layer_norm(torch.zeros((), device="cuda")),
                lambda: training.layer_norm_grad(x[:3], x, s, s), lambda: training.layer_norm_grad(x.half(), x, s, s),
                lambda: training.layer_norm_grad(x, x, s[:3], s), lambda: training.layer_norm_grad(x, x, s, s.double()),
                lambda: training.layer_norm_grad(x, x, s, s, d_sum=x.half())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: training.layer_norm(x.double()), lambda: training.layer_norm(x, w.cpu())):
        with pytest.raises(TypeError):
            bad()
