"""Rows of an embedding table and their gradient (tcc_amd.training over
include/tcc_training.h) against plain 64-bit evaluations.

The lookup is one fp32 product rounded once, so it is compared bit for bit.
The gradient of a row with m terms is a sum in fp32: whatever the order, its
error is below (m + 2) 2^-24 times scale * sum |terms| (m - 1 additions, the
scale's rounding and the product's), plus one rounding to the output's type
(2^-24, 2^-8, 2^-11 of the result; fp16 below 2^-14 rounds to 2^-25)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U_OUT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def ids_of(kind, n, V, gen):
    if kind == "uniform":
        return torch.randint(0, V, (n,), generator=gen)
    if kind == "hubs":
        return (torch.rand(n, generator=gen, dtype=torch.float64) ** 4 * V).long().clamp_(max=V - 1)
    if kind == "one":
        return torch.full((n,), V - 1)
    if kind == "ordered":
        return torch.arange(n) % V
    raise ValueError(kind)


def grad64(d, ids, V, scale, padding=None):
    """(sum, sum of magnitudes, terms) of every row in 64 bits."""
    d = d.double().cpu()
    keep = (ids >= 0) & (ids < V)
    if padding is not None:
        keep &= ids != padding
    d, ids = d[keep], ids[keep].long()
    s = torch.zeros((V, d.shape[1]), dtype=torch.float64).index_add_(0, ids, d)
    m = torch.zeros((V, d.shape[1]), dtype=torch.float64).index_add_(0, ids, d.abs())
    return s * scale, m * scale, torch.bincount(ids, minlength=V).double().unsqueeze(1)


def check_grad(got, d, ids, V, scale, padding=None, base=None):
    want, mag, terms = grad64(d, ids.cpu(), V, scale, padding)
    extra = 0.0
    if base is not None:
        b = base.double().cpu()
        want, extra = want + b, 2.0**-24 * (want.abs() + b.abs())
    tol = (terms + 2) * 2.0**-24 * mag + extra
    tol = tol + U_OUT[got.dtype] * (want.abs() + tol) + (2.0**-25 if got.dtype == torch.float16 else 0.0)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), f"largest excess {float((err - tol).max()):.3e}"
    untouched = (terms == 0).expand_as(want)
    keep = torch.zeros_like(want) if base is None else base.double().cpu()
    assert torch.equal(got.double().cpu()[untouched], keep[untouched])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,n,D", [(1, 1, 1), (5, 1, 7), (300, 1000, 32), (4096, 777, 100), (50, 3001, 33), (9, 257, 602),
                                   (2000, 64, 8), (33, 129, 1030)])
def test_lookup_bit_for_bit(gpu, dtype, V, n, D):
    from tcc_amd import training

    gen = torch.Generator().manual_seed(V * 31 + n + D)
    table = torch.randn((V, D), generator=gen).to(dtype).cuda()
    for width, pad in ((torch.int32, None), (torch.int64, V // 2)):
        ids = torch.randint(0, V, (n,), generator=gen).to(width).cuda()
        got = training.embedding_lookup(table, ids, scale=1.7, padding_idx=pad)
        want = (table[ids.long()].float() * 1.7).to(dtype)
        if pad is not None:
            want[ids == pad] = 0
        assert torch.equal(got, want)


def test_lookup_strides_shapes_and_out(gpu):
    from tcc_amd import training

    wide = torch.randn((500, 90), device="cuda")
    ids = torch.randint(0, 500, (6, 11), device="cuda")
    for cols in (slice(0, 64), slice(3, 40), slice(1, 2)):  # 16-byte rows, odd offsets, one column
        table = wide[:, cols]
        assert torch.equal(training.embedding_lookup(table, ids), table[ids])
        room = torch.full((40, 77), 5.0, device="cuda")
        flat = ids[:3].reshape(-1)
        out = room[:33, 4:4 + table.shape[1]]
        assert training.embedding_lookup(table, flat, scale=0.5, out=out) is out
        assert torch.equal(out, table[flat] * 0.5)
        rest = room.clone()
        rest[:33, 4:4 + table.shape[1]] = 5.0
        assert bool((rest == 5.0).all()), "written outside the output"
    t = wide.t()  # columns contiguous: copied
    assert torch.equal(training.embedding_lookup(t, ids % 90), t[ids % 90])
    assert training.embedding_lookup(wide, ids[:0]).shape == (0, 11, 90)
    # every second id: not contiguous
    assert torch.equal(training.embedding_lookup(wide, ids[:, ::2]), wide[ids[:, ::2]])


def test_lookup_refused_ids_and_non_finite_rows(gpu):
    from tcc_amd import swtcf, training

    table = torch.randn((10, 12), device="cuda")
    table[3], table[4, 5] = float("inf"), float("nan")
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    ids = torch.tensor([3, 4, 9], device="cuda")
    got = training.embedding_lookup(table, ids, scale=2.0, device_error=word, padding_idx=3)
    assert torch.equal(got[0], torch.zeros(12, device="cuda")) and bool(got[1].isnan().sum() == 1)
    assert int(word) == 0
    for bad in (-1, 10, 1 << 40, -(1 << 40)):
        word.zero_()
        got = training.embedding_lookup(table, torch.tensor([1, bad, 2], device="cuda"), device_error=word)
        assert torch.equal(got, torch.stack([table[1], torch.zeros(12, device="cuda"), table[2]]))
        assert int(word) == swtcf.DEVERR_FEATURE_INDEX
        word.zero_()
        d = torch.randn((3, 12), device="cuda")
        d[1] = float("nan")  # the refused row is not read
        g = training.embedding_grad(d, torch.tensor([1, bad, 2], device="cuda"), 10, device_error=word)
        assert torch.equal(g[1], d[0]) and torch.equal(g[2], d[2]) and int((g != 0).any(1).sum()) == 2
        assert int(word) == swtcf.DEVERR_FEATURE_INDEX


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["uniform", "hubs", "one", "ordered"])
@pytest.mark.parametrize("V,n,D", [(1, 1, 1), (7, 2, 5), (300, 1000, 32), (4096, 777, 100), (50, 3001, 33), (9, 4097, 130),
                                   (70_000, 20_011, 16), (100, 70_000, 20), (40, 300, 602),
                                   (5_000_000, 5001, 2), (2047, 65_536, 3), (2048, 65_537, 3), (3, 3000, 9), (60, 40_000, 36)])
def test_grad(gpu, dtype, kind, V, n, D):
    from tcc_amd import training

    gen = torch.Generator().manual_seed(V + 7 * n + D)
    ids = ids_of(kind, n, V, gen).to(torch.int32 if D % 2 else torch.int64)
    d = torch.randn((n, D), generator=gen).to(dtype).cuda()
    pad = int(ids[0]) if kind == "hubs" and V > 1 else None
    if pad is not None:
        d[(ids == pad).cuda()] = float("nan")  # padding rows count for nothing, whatever they hold
    got = training.embedding_grad(d, ids.cuda(), V, scale=0.25, padding_idx=pad)
    check_grad(got, d.nan_to_num(), ids, V, 0.25, pad)
    again = training.embedding_grad(d, ids.cuda(), V, scale=0.25, padding_idx=pad)
    assert torch.equal(got, again), "the same inputs give the same bits"


@pytest.mark.parametrize("dtype", TYPES)
def test_grad_accumulates_into_rows_that_occur(gpu, dtype):
    from tcc_amd import training

    gen = torch.Generator().manual_seed(3)
    V, n, D = 5000, 900, 48
    ids = ids_of("hubs", n, V, gen).cuda()
    d = torch.randn((n, D), generator=gen).to(dtype).cuda()
    room = torch.randn((V, 64), generator=gen).to(dtype).cuda()
    grad = room[:, 8:8 + D]
    base = grad.clone()
    assert training.embedding_grad(d, ids, V, scale=3.0, grad=grad, accumulate=True) is grad
    check_grad(grad, d, ids, V, 3.0, base=base)
    # and rows of a wider buffer are written without touching the rest
    rest = torch.cat([room[:, :8], room[:, 8 + D:]], 1).clone()
    training.embedding_grad(d, ids, V, grad=grad)
    check_grad(grad, d, ids, V, 1.0)
    assert torch.equal(rest, torch.cat([room[:, :8], room[:, 8 + D:]], 1))


def test_grad_without_ids(gpu):
    from tcc_amd import training

    none = torch.empty(0, dtype=torch.int64, device="cuda")
    g = training.embedding_grad(torch.empty((0, 6), device="cuda"), none, 40)
    assert torch.equal(g, torch.zeros((40, 6), device="cuda"))
    g.fill_(2.0)
    training.embedding_grad(torch.empty((0, 6), device="cuda"), none, 40, grad=g, accumulate=True)
    assert bool((g == 2.0).all())
    # every id is padding
    pad = torch.full((33,), 4, dtype=torch.int32, device="cuda")
    g = training.embedding_grad(torch.ones((33, 6), device="cuda"), pad, 40, padding_idx=4)
    assert torch.equal(g, torch.zeros((40, 6), device="cuda"))


def test_grad_of_broadcast_and_transposed_rows(gpu):
    """d_out as sums give it: one row for all (stride 0), or column-major."""
    from tcc_amd import training

    ids = torch.randint(0, 30, (200,), device="cuda")
    one = torch.randn((1, 24), device="cuda").expand(200, 24)
    check_grad(training.embedding_grad(one, ids, 30), one, ids, 30, 1.0)
    cols = torch.randn((24, 200), device="cuda").t()
    check_grad(training.embedding_grad(cols, ids, 30), cols, ids, 30, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V", [(200_000, 3000), (600_000, 400_000), (1_000_003, 70)])
@pytest.mark.parametrize("D", [1, 4, 8, 33])
def test_grad_of_long_lists(gpu, dtype, n, V, D):
    """Chunks of 16 and 64 rows, with the most keys a workgroup can hold where
    a row is one vector; hubs of many parts; accumulated too."""
    from tcc_amd import training

    gen = torch.Generator().manual_seed(n + D)
    ids = ids_of("hubs", n, V, gen).to(torch.int32)
    d = torch.randn((n, D), generator=gen).to(dtype).cuda()
    got = training.embedding_grad(d, ids.cuda(), V, scale=0.5)
    check_grad(got, d, ids, V, 0.5)
    assert torch.equal(got, training.embedding_grad(d, ids.cuda(), V, scale=0.5))
    base = torch.randn((V, D), generator=gen).to(dtype).cuda()
    check_grad(training.embedding_grad(d, ids.cuda(), V, scale=0.5, grad=base.clone(), accumulate=True), d, ids, V, 0.5,
               base=base)


@pytest.mark.parametrize("n,D,dtype", [(700_003, 101, torch.float32), (600_001, 232, torch.bfloat16)])
def test_lookup_past_the_caches(gpu, n, D, dtype):
    """Outputs larger than the last level of cache (256 MB)."""
    from tcc_amd import training

    gen = torch.Generator(device="cuda").manual_seed(D)
    table = torch.randn((5000, D), generator=gen, device="cuda").to(dtype)
    ids = torch.randint(0, 5000, (n,), generator=gen, device="cuda")
    got = training.embedding_lookup(table, ids, scale=0.3, padding_idx=7)
    want = (table[ids].float() * 0.3).to(dtype)
    want[ids == 7] = 0
    assert torch.equal(got, want)


def test_places_past_32_bits(gpu):
    """A table of over 2^32 elements: its last rows, and their gradient."""
    from tcc_amd import training

    V, D = 2_200_000, 2000  # 4.4e9 elements
    table = torch.empty((V, D), dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([V - 1, 0, V - 2, V - 1], device="cuda")
    table[ids] = torch.randn((4, D), device="cuda").to(torch.bfloat16)
    assert torch.equal(training.embedding_lookup(table, ids), table[ids])
    d = torch.randn((4, D), device="cuda").to(torch.bfloat16)
    table[ids] = 0
    training.embedding_grad(d, ids, V, grad=table, accumulate=True)
    assert torch.equal(table[0], d[1]) and torch.equal(table[V - 2], d[2])
    assert torch.equal(table[V - 1], (d[0].float() + d[3].float()).to(torch.bfloat16))
    g = training.embedding_grad(d, ids, V, grad=table)
    assert torch.equal(g[V - 2], d[2]) and int(torch.count_nonzero(g[V - 3])) == 0


def test_lookup_of_more_than_a_launch(gpu):
    """17.3e9 elements that lanes take one by one (35 GB): more than one launch
    has threads for, with the launches' ends inside rows."""
    from tcc_amd import training

    V, n, D = 1000, 171_000_007, 101
    gen = torch.Generator(device="cuda").manual_seed(8)
    table = torch.randn((V, D), generator=gen, device="cuda").to(torch.float16)
    ids = torch.randint(0, V, (n,), generator=gen, device="cuda", dtype=torch.int32)
    got = training.embedding_lookup(table, ids)
    for at in range(0, n, 10_000_000):
        assert torch.equal(got[at:at + 10_000_000], table[ids[at:at + 10_000_000].long()])


@pytest.mark.parametrize("n", [50, 5000, 70_000])
def test_grad_of_the_longest_table(gpu, n):
    """2^32 - 2 rows of one fp16 element: ids at both ends and between, every
    other row zeroed, the last windows' too."""
    from tcc_amd import training

    V = 2**32 - 2
    gen = torch.Generator().manual_seed(n)
    ids = torch.cat([torch.randint(0, V, (n - 6,), generator=gen), torch.tensor([0, 3, V - 20, V - 9, V - 9, V - 5])]).cuda()
    d = torch.ones((n, 1), dtype=torch.float16, device="cuda")
    grad = torch.full((V, 1), 7.0, dtype=torch.float16, device="cuda")
    training.embedding_grad(d, ids, V, grad=grad)
    rows, count = torch.unique(ids, return_counts=True)
    assert torch.equal(grad[rows, 0], count.to(torch.float16))
    assert sum(int(torch.count_nonzero(grad[at:at + 2**29])) for at in range(0, V, 2**29)) == rows.numel()


def test_columns_past_32_bits_are_refused(gpu):
    """Tables without a row, so that nothing of that width is in memory."""
    from tcc_amd import training

    none = torch.empty(0, dtype=torch.int64, device="cuda")
    wide = torch.empty((0, 2**32 + 8), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        training.embedding_lookup(wide, none)
    with pytest.raises(ValueError):
        training.embedding_grad(wide, none, 0)


def test_gradient_against_differences(gpu):
    """<grad, e> is the change of sum(w * lookup) along e: the lookup is
    linear, so the difference quotient is exact up to rounding."""
    from tcc_amd import training

    gen = torch.Generator().manual_seed(9)
    V, n, D = 120, 500, 40
    ids = ids_of("hubs", n, V, gen).cuda()
    w = torch.randn((n, D), generator=gen).cuda()
    table, e = torch.randn((V, D), generator=gen).cuda(), torch.randn((V, D), generator=gen).cuda()
    f = lambda t: (training.embedding_lookup(t, ids, scale=1.5).double() * w.double()).sum()  # noqa: E731
    along = float((training.embedding_grad(w, ids, V, scale=1.5).double() * e.double()).sum())
    quotient = float((f(table + e) - f(table - e)) / 2)
    size = float((1.5 * w.abs().double() * (table.abs() + e.abs()).double()[ids]).sum())
    assert abs(along - quotient) <= 8 * 2.0**-24 * size


def test_replayed_graph_and_other_stream(gpu):
    from tcc_amd import training

    gen = torch.Generator(device="cuda").manual_seed(5)
    V, n, D = 3000, 5000, 36
    ids = torch.randint(0, V, (n,), generator=gen, device="cuda")
    table = torch.randn((V, D), generator=gen, device="cuda")
    d = torch.randn((n, D), generator=gen, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = training.embedding_lookup(table, ids, stream=side)
    b = training.embedding_grad(d, ids, V, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, table[ids]) and torch.equal(b, training.embedding_grad(d, ids, V))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = training.embedding_lookup(table, ids)
        b = training.embedding_grad(d, ids, V)
    for _ in range(3):
        ids.copy_(torch.randint(0, V, (n,), generator=gen, device="cuda"))
        d.copy_(torch.randn((n, D), generator=gen, device="cuda"))
        want = training.embedding_grad(d, ids, V)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, table[ids]) and torch.equal(b, want)
