"""The streamed paths of tcc_amd.training.top_logits: a wave a row where there are
many, a workgroup a row else, over rows of every order.  The bounds of
test_gpu_top_logits.py, whose terms that grow with the row are left out: a rest is
off by 4 u |rest| + T u (64 + 4 log C)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def many():
    """Rows from which on a wave takes each."""
    return 12 * torch.cuda.get_device_properties(0).multi_processor_count


def rows_of(kind, n, C, dtype, gen):
    if kind == "random":
        return torch.empty((n, C), device="cuda").normal_(0.0, 3.0, generator=gen).to(dtype)
    if kind == "up":
        return torch.linspace(-9.0, 9.0, C, device="cuda").to(dtype).expand(n, C).contiguous()
    if kind == "equal":
        z = torch.ones((n, C), dtype=dtype, device="cuda")
        z[:, torch.randint(0, C, (9,), generator=gen, device="cuda")] = 2.0
        return z
    z = torch.empty((n, C), device="cuda").normal_(generator=gen)
    if kind == "masked":  # five of each row are left
        keep = torch.rand((n, C), generator=gen, device="cuda").topk(5, dim=1).indices
        return torch.full_like(z, -np.inf).scatter_(1, keep, z.gather(1, keep)).to(dtype)
    if kind == "masked parts":  # what a wave, a batch or the end of a row has
        z[::3, : C // 2] = -np.inf
        z[1::3, 64:] = -np.inf
        z[2::3, : C - 70] = -np.inf
        return z.to(dtype)
    z[:, ::97] = np.nan  # "nan"
    z[::2, C // 3] = np.inf
    return z.to(dtype)


def check(z, K, T, rows):
    from tcc_amd import training

    values, ids, rest = training.top_logits(z, K, temperature=T)
    C = z.shape[1]
    for i in rows:
        v = z[i].double()
        # a NaN above all, the lowest class first among equals
        want = torch.sort(v + 0.0, descending=True, stable=True).indices[:K]
        assert torch.equal(ids[i].long(), want), f"row {i}"
        assert torch.equal(values[i].nan_to_num(6e4, 5e4, -5e4), z[i, want].nan_to_num(6e4, 5e4, -5e4))
        left = v.clone()
        left[want] = -np.inf
        right = float(torch.logsumexp(left / T, 0) * T)
        if not np.isfinite(right):
            assert np.array_equal(float(rest[i]), right, equal_nan=True)
        else:
            assert abs(float(rest[i]) - right) <= 4 * U * abs(right) + T * U * (64 + 4 * np.log(C))


KINDS = ["random", "up", "equal", "masked", "masked parts", "nan"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("C,K", [(4097, 1), (9000, 17), (30_001, 32)])
def test_a_wave_a_row(gpu, dtype, kind, C, K):
    gen = torch.Generator(device="cuda").manual_seed(C)
    n = many() + 5
    z = rows_of(kind, n, C, dtype, gen)
    check(z, K, 2.0, [0, 1, 2, 3, n // 2, n - 2, n - 1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,C,K", [(7, 4097, 1), (6, 4609, 64), (300, 9217, 7), (6, 33_000, 64), (3, 100_003, 17),
                                   (2, 1_000_001, 64), (1, 3_000_000, 32)])
def test_a_workgroup_a_row(gpu, dtype, kind, n, C, K):
    """The last batch of some waves only, too."""
    gen = torch.Generator(device="cuda").manual_seed(C)
    z = rows_of(kind, n, C, dtype, gen)
    check(z, K, 1.5, sorted({0, min(1, n - 1), min(2, n - 1), n // 2, n - 1}))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batches", [2, 5])
@pytest.mark.parametrize("waves", [1, 2, 3, 4])
def test_ends_where_some_waves_have_no_batch(gpu, dtype, batches, waves):
    """Rows that end inside the batch before which four waves agree anew."""
    V = 16 // dtype.itemsize
    C = batches * 4 * 256 * V + (waves - 1) * 64 * V + 3
    gen = torch.Generator(device="cuda").manual_seed(C)
    for K in (3, 64):
        check(rows_of("random", 5, C, dtype, gen), K, 1.0, range(5))


@pytest.mark.parametrize("dtype", TYPES)
def test_the_largest_in_one_waves_part(gpu, dtype):
    """A bound from one wave alone would leave out what the others' lack."""
    V = 16 // dtype.itemsize
    C = 40 * 4 * 64 * V * 4
    z = torch.zeros((4, C), dtype=dtype, device="cuda")
    for w in range(4):
        z[w].view(-1, 4, 64 * V)[:, w, 5] = torch.linspace(1.0, 60.0, C // (4 * 64 * V), device="cuda").to(dtype)
    for K in (1, 9, 40, 64):
        check(z, K, 1.0, range(4))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,K", [(1, 64), (1, 5), (0, 32)])
def test_rising_rows(gpu, dtype, n, K):
    """Logits whose level rises along the row: every bound is soon too low."""
    n, C = n or many(), 200_000 if n else 20_000
    gen = torch.Generator(device="cuda").manual_seed(K)
    z = torch.empty((n, C), device="cuda").normal_(generator=gen).add_(torch.linspace(0.0, 12.0, C, device="cuda")).to(dtype)
    check(z, K, 1.0, [0, n // 2, n - 1])
