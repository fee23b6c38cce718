"""The top logits of every row (tcc_amd.training.top_logits) against sorts, and
the logit of the rest against 64-bit sums.

Values and ids are equal bits.  The rest is m + T log(s), s the sum of
e = exp((z - m) / T): an exponent x = (z - m) / T has three roundings
(u = 2^-24 each), and the mean of |x| over the shares is at most log C (their
entropy, log s + that mean, is), so s is off by 3 u log C of itself; its C terms
are added over 64 lanes at least, C / 64 + 100 roundings with the rescalings,
merges and the steps over the lanes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1, 1), (3, 2, 1), (5, 2, 2), (9, 3, 2), (64, 7, 7), (40, 8, 3), (130, 33, 16), (300, 47, 4), (77, 64, 64),
          (101, 100, 8), (60, 127, 1), (60, 257, 64), (20, 1001, 33), (13, 4096, 64), (9, 4097, 5), (7, 20_000, 64),
          (5, 50_001, 32), (3, 140_000, 48)]


def check(got, z, K, T):
    values, ids, rest = got
    n, C = z.shape
    v = z.double().cpu() + 0.0
    want = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :K]
    assert ids.dtype == torch.int32 and torch.equal(ids.cpu().long(), want)
    picked = z.cpu().gather(1, want)
    assert values.dtype == z.dtype
    assert torch.equal(values.cpu().nan_to_num(7e4, 6e4, -6e4), picked.nan_to_num(7e4, 6e4, -6e4))
    left = torch.logsumexp(v.scatter(1, want, -np.inf) / T, 1) * T
    if K == C:
        assert bool((rest == -np.inf).all())
        return
    finite = torch.isfinite(left)
    assert torch.equal(rest.double().cpu()[~finite].nan_to_num(7.0), left[~finite].nan_to_num(7.0))
    tol = 4 * U * left.abs() + T * U * (3 * np.log(C) + C / 64 + 100)
    assert bool(((rest.double().cpu() - left).abs() <= tol)[finite].all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,C,K", SHAPES)
def test_random_rows(gpu, dtype, n, C, K):
    from tcc_amd import training

    gen = torch.Generator().manual_seed(n + C)
    for spread, T in ((3.0, 1.0), (40.0, 3.0)):
        z = (torch.randn((n, C), generator=gen) * spread).to(dtype).cuda()
        got = training.top_logits(z, K, temperature=T)
        check(got, z, K, T)
        for p, q in zip(got, training.top_logits(z, K, temperature=T)):
            assert torch.equal(p, q), "the same inputs give the same bits"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,C,K", [(500, 100, 16), (200, 100, 64), (300, 300, 40), (300, 511, 64), (200, 513, 64), (120, 700, 64),
                                   (90, 1500, 50), (700, 1025, 3), (40, 3000, 16), (1500, 4100, 8), (300, 8193, 64),
                                   (30, 40_000, 40)])
def test_more_of_every_path(gpu, dtype, n, C, K):
    """Random rows; rows whose elements are nearly all masked; equal ones with
    a few others."""
    from tcc_amd import training

    gen = torch.Generator().manual_seed(n + C)
    z = torch.randn((n, C), generator=gen) * 3
    z[n // 4:n // 2] = -np.inf
    z[n // 4:n // 2, torch.randperm(C, generator=gen)[:5]] = torch.randn(5, generator=gen)
    z[n // 2:3 * n // 4] = 1.0
    z[n // 2:3 * n // 4, torch.randperm(C, generator=gen)[:9]] = torch.randn(9, generator=gen) + 1
    z = z.to(dtype).cuda()
    check(training.top_logits(z, K, temperature=2.0), z, K, 2.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [5, 40, 300, 4000, 9000])
@pytest.mark.parametrize("levels", [1, 2, 7])
def test_ties_go_to_the_lowest_class(gpu, dtype, C, levels):
    from tcc_amd import training

    gen = torch.Generator().manual_seed(C)
    z = (torch.randint(0, levels, (30, C), generator=gen) - levels // 2).to(dtype)
    z[::2] *= -1.0  # zeros of both signs are equal
    z = z.cuda()
    for K in sorted({1, 2, min(C, 17), min(C, 64)}):
        check(training.top_logits(z, K), z, K, 1.0)


@pytest.mark.parametrize("order", ["up", "down"])
@pytest.mark.parametrize("C", [64, 200, 4096, 30_000])
def test_sorted_rows(gpu, order, C):
    """Every element beats those before it, or none does."""
    from tcc_amd import training

    z = torch.linspace(-9.0, 9.0, C).repeat(3, 1)
    z = (z if order == "up" else z.flip(1)).contiguous().cuda()
    for K in (1, 20, 64):
        check(training.top_logits(z, K, temperature=2.0), z, K, 2.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [6, 70, 500, 6000])
def test_infinities_and_nan(gpu, dtype, C):
    from tcc_amd import training

    gen = torch.Generator().manual_seed(C)
    z = torch.randn((12, C), generator=gen)
    z[0] = -np.inf  # nothing but masked classes
    z[1, 1:] = -np.inf
    z[2, C // 2:] = -np.inf
    z[3, 4] = np.inf
    z[4, :5] = np.inf
    z[5, 3] = np.nan
    z[6, :6] = np.nan
    z[7, 2], z[7, 5] = np.nan, np.inf
    z[8] = torch.finfo(dtype).min
    z[9] = torch.finfo(dtype).max
    z = z.to(dtype).cuda()
    for K in (1, 3, 6):
        check(training.top_logits(z, K), z, K, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignments(gpu, dtype):
    from tcc_amd import training

    gen = torch.Generator().manual_seed(3)
    x = torch.randn((40, 6000), generator=gen).to(dtype).cuda()
    for cols in (slice(1, 48), slice(3, 500), slice(5, 5998), slice(0, 4)):
        K = min(9, cols.stop - cols.start)
        check(training.top_logits(x[:, cols], K), x[:, cols], K, 1.0)
    turned = x[:, :99].t().contiguous().t()
    check(training.top_logits(turned, 5), turned, 5, 1.0)


def test_no_rows_and_many(gpu):
    from tcc_amd import training

    values, ids, rest = training.top_logits(torch.empty((0, 9), device="cuda"), 4)
    assert values.shape == ids.shape == (0, 4) and rest.shape == (0,)
    z = torch.randn((200_003, 20), device="cuda")
    check(training.top_logits(z, 3), z, 3, 1.0)


@pytest.mark.parametrize("T", [1e-18, 1e-4, 1e4, 1e18])
@pytest.mark.parametrize("C", [9, 150, 700, 6000])
def test_extreme_temperatures(gpu, C, T):
    from tcc_amd import training

    z = torch.randn((50, C), generator=torch.Generator().manual_seed(C)).cuda()
    T = float(np.float32(T))
    check(training.top_logits(z, 4, temperature=T), z, 4, T)


def test_places_past_32_bits(gpu):
    """4.5e9 logits: the last rows'."""
    from tcc_amd import training

    z = torch.empty((90_000, 50_000), dtype=torch.bfloat16, device="cuda").normal_()
    values, ids, rest = training.top_logits(z, 12)
    end = slice(90_000 - 20, 90_000)
    check((values[end], ids[end], rest[end]), z[end], 12, 1.0)


def test_replayed_graph_and_other_stream(gpu):
    from tcc_amd import training

    gen = torch.Generator().manual_seed(4)
    for C in (90, 7000):
        z = torch.randn((500, C), generator=gen).cuda()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = training.top_logits(z, 10, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        check(got, z, 10, 1.0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = training.top_logits(z, 10)
        for _ in range(3):
            z.copy_(torch.randn(z.shape, generator=gen))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for p, q in zip(out, training.top_logits(z, 10)):
                assert torch.equal(p, q)


def test_refusals_on_the_device(gpu):
    from tcc_amd import training

    z = torch.zeros((4, 100), device="cuda")
    for bad in (lambda: training.top_logits(z, 0), lambda: training.top_logits(z, 65), lambda: training.top_logits(z[:, :5], 6),
                lambda: training.top_logits(z, 3, temperature=0.0), lambda: training.top_logits(z, 3, temperature=float("nan")),
                lambda: training.top_logits(z[0], 3), lambda: training.top_logits(z[:, :0], 1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        training.top_logits(z.double(), 3)
