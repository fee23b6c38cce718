"""Rows of very many classes: the softmax sums of tcc_amd.training.distill_loss
keep their digits however long a row is.

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
