"""Rows of very many classes: the softmax sums of tcc_amd.training.distill_loss
and the rest of top_logits keep their digits however long a row is.

Bounds, with u = 2^-24 and x = (z - m) / T, none of which grows with the row: an
exponent has four roundings of |x| (the factor log2(e) / T, the difference, the
product and the change of the maximum) and the instruction one ulp, the terms of
a batch are added 32 at most in 32 bits and the batches in 64, the lanes in ten
steps: a sum is off by (64 + 4 mean |x|) u of itself, the mean over its shares."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
U_OUT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}
BY_DTYPE = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])


def share(row, T, without=()):
    """(maximum, sum of exp((z - maximum) / T), mean of |x| over the shares) of a
    row but for some of its classes, in 64 bits."""
    without = list(without)
    top = float(row.max()) if not without else float(row.index_fill(0, torch.tensor(without, device="cuda"), -np.inf).max())
    s = mean = 0.0
    for part in row.split(1 << 25):
        x = (part.double() - top) / T
        s += float(x.exp().sum())
        mean += float((x.abs() * x.exp()).sum())
    for c in without:
        x = (float(row[c]) - top) / T
        s -= math.exp(x)
        mean -= abs(x) * math.exp(x)
    return top, s, mean / s


def check_loss(row, ids, T):
    """Loss, stats and gradient of one row against entries at `ids`."""
    from tcc_amd import training

    z, C = row[None], row.numel()
    values = torch.linspace(1.0, 0.0, len(ids), device="cuda")[None].to(row.dtype)
    at = torch.tensor([ids], dtype=torch.int32, device="cuda")
    m, s, mean = share(row, T)
    mr, sr, mean_r = share(row, T, ids)
    tol, tol_r = (64 + 4 * mean) * U, (64 + 4 * mean_r) * U
    picked = row[at[0].long()].double().cpu()
    for rest in (None, torch.full((1,), 2.0, device="cuda")):
        loss, stats, _ = training.distill_loss(z, values, at, rest=rest, temperature=T)
        assert float(stats[0, 0]) == m and abs(float(stats[0, 1]) / s - 1) <= tol
        t, log_q = values[0].double().cpu(), (picked - m) / T - math.log(s)
        if rest is not None:
            assert float(stats[0, 2]) == mr and abs(float(stats[0, 3]) / sr - 1) <= tol_r
            t = torch.cat([t, torch.tensor([2.0]).double()])
            log_q = torch.cat([log_q, torch.tensor([(mr - m) / T + math.log(sr / s)])])
        log_p = torch.log_softmax(t / T, 0)
        p = log_p.exp()
        want = T * T * float((p * (log_p - log_q)).sum())
        spread = float((p * (log_p.abs() + log_q.abs())).sum()) + math.log(s)
        assert abs(float(loss) - want) <= T * T * (tol + tol_r + 8 * U * spread)
        dz = training.distill_grad(torch.ones((), device="cuda"), z, values, at, stats, rest=rest, temperature=T)[0]
        # the classes without an entry have c T q, q = exp(x) / s; c is a difference of two sums' quotients
        c = 1.0 if rest is None else 1.0 - float(p[-1]) * s / (sr * math.exp((mr - m) / T))
        err = tol if rest is None else (tol + tol_r) * (1 + abs(c - 1))
        for part in (slice(0, 1 << 20), slice(C // 2, C // 2 + (1 << 20)), slice(C - (1 << 20), C)):
            x = (row[part].double() - m) / T
            q = x.exp() * (T / s)
            off = q * (abs(c) * U * (4 * (x.abs() + (m - mr) / T) + 16) + err)
            off = off + U_OUT[row.dtype] * (abs(c) * q + off) + 1e-37
            off[[i - part.start for i in ids if part.start <= i < part.stop]] = np.inf
            assert bool(((dz[part].double() - c * q).abs() <= off).all())
        # the entries' classes T (q - p)
        x = (picked - m) / T
        q, mine = x.exp() / s, p[:len(ids)]
        off = T * (q * (tol + 4 * U * x.abs()) + mine * 32 * U)
        off = off + U_OUT[row.dtype] * (T * (q - mine).abs() + off) + 1e-37
        assert bool(((dz[at[0].long()].double().cpu() - T * (q - mine)).abs() <= off).all())


@BY_DTYPE
@pytest.mark.parametrize("T", [1.0, 4.0])
def test_loss_of_equal_logits_below_one_maximum(gpu, dtype, T):
    C = 1 << 28
    row = torch.full((C,), -1.25, dtype=dtype, device="cuda")
    row[C // 3] = 0.0
    check_loss(row, [C // 3, 7, C - 1], T)


@BY_DTYPE
def test_loss_of_random_logits(gpu, dtype):
    C = (1 << 27) + 11
    row = torch.empty(C, dtype=dtype, device="cuda").normal_(0.0, 3.0, generator=torch.Generator(device="cuda").manual_seed(1))
    check_loss(row, [5, 1000, C - 2], 2.0)


@pytest.mark.parametrize("ends", [(-9.0, 9.0), (9.0, -9.0), (-0.5, 0.25)])
def test_loss_of_sorted_logits(gpu, ends):
    """The maximum rises with every batch, by little: the sums before it are not
    rounded again each time."""
    row = torch.linspace(*ends, 1 << 27, device="cuda")
    check_loss(row, [0, 1 << 26, (1 << 27) - 1], 1.0)


def check_rest(z, K, T, others):
    """The rest of row 0 against the (value, count) of all classes that are not
    taken; the rows are equal."""
    from tcc_amd import training

    values, ids, rest = training.top_logits(z, K, temperature=T)
    m = max(v for v, _ in others)
    s = sum(n * math.exp((v - m) / T) for v, n in others)
    mean = sum(n * (m - v) / T * math.exp((v - m) / T) for v, n in others) / s
    want = m + T * math.log(s)
    assert bool((rest == rest[0]).all())
    # log2 and its product with T log 2 round to two ulps each of what they give
    assert abs(float(rest[0]) - want) <= T * (64 + 4 * mean) * U + 4 * U * (abs(m) + T * math.log(s))
    return values, ids


@BY_DTYPE
def test_rest_of_a_streamed_row(gpu, dtype):
    """A workgroup's row: each of its waves has one class at the bound."""
    C, V = 1 << 28, 16 // dtype.itemsize
    z = torch.full((1, C), -1.25, dtype=dtype, device="cuda")
    high = [w * 64 * V for w in range(4)]
    z[0, 1:256 * V:V] = 0.0  # the largest of each lane's rest
    z[0, high] = 0.5
    values, ids = check_rest(z, 1, 1.0, [(0.5, 3), (0.0, 256), (-1.25, C - 260)])
    assert ids.tolist() == [[0]] and values.tolist() == [[0.5]]
    values, ids = check_rest(z, 4, 2.0, [(0.0, 256), (-1.25, C - 260)])
    assert ids.tolist() == [high]


@BY_DTYPE
def test_rest_of_rows_streamed_by_waves(gpu, dtype):
    """A wave a row, where there are many: each of its lanes has a class at the bound."""
    n = 12 * torch.cuda.get_device_properties(0).multi_processor_count
    C, V = 1 << 20, 16 // dtype.itemsize
    z = torch.full((n, C), -1.25, dtype=dtype, device="cuda")
    z[:, 1:64 * V:V] = 0.0
    z[:, :64 * V:V] = 0.5
    values, ids = check_rest(z, 17, 1.0, [(0.5, 64 - 17), (0.0, 64), (-1.25, C - 128)])
    assert bool((values == 0.5).all()) and bool((ids == torch.arange(0, 17 * V, V, device="cuda")).all())


@BY_DTYPE
def test_rest_of_a_row_of_equal_logits(gpu, dtype):
    """More classes at the bound than there is room for."""
    C = 1 << 26
    z = torch.full((1, C), -1.25, dtype=dtype, device="cuda")
    z[0, C // 2] = 3.0
    _, ids = check_rest(z, 3, 1.0, [(-1.25, C - 3)])
    assert ids.tolist() == [[C // 2, 0, 1]]


@pytest.mark.parametrize("ends", [(-9.0, 9.0), (-0.5, 0.25)])
def test_rest_of_a_sorted_row(gpu, ends):
    """Every class beats those before it."""
    from tcc_amd import training

    row = torch.linspace(*ends, 1 << 24, device="cuda")
    values, ids, rest = training.top_logits(row[None], 5)
    order = torch.sort(row[-2000:], descending=True, stable=True)
    assert torch.equal(ids[0].long(), order.indices[:5] + row.numel() - 2000)
    m, s, mean = share(row, 1.0, ids[0].tolist())
    assert abs(float(rest) - m - math.log(s)) <= (64 + 4 * mean) * U + 4 * U * (abs(m) + math.log(s))
