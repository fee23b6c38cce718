"""How many digits the layer norm's parameter gradients keep over many rows.

With u = 2^-24, a rounding is off by at most u |s|, u / sqrt(3) in the root mean
square.  A run of n rows is summed in 32 bits: terms of either sign leave its sum
off by u sqrt(n / 6) of itself, as a mean; a term has three roundings of its own
(xh two, its product one) and the workgroups' sums and the result one each:
u sqrt(5 / 3).  Runs are of 8 to 15 rows of fp32, of 12 to 23 of 16 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,C", [(1_000_000, 256), (6_000_000, 40), (400_000, 384), (500_000, 512), (200_000, 700),
                                 (300_000, 1000), (5_000_000, 6), (3_000_000, 13), (1_000_000, 100), (60_000, 2000),
                                 (30_000, 4096), (20_000, 8000)])
@pytest.mark.parametrize("dtype,run", [(torch.float32, 15), (torch.bfloat16, 23)])
def test_parameter_gradients(gpu, dtype, run, N, C):
    from tcc_amd import training

    gen = torch.Generator(device="cuda").manual_seed(C)
    x, d = torch.randn((2, N, C), generator=gen, device="cuda").to(dtype)
    w, b = torch.rand((2, C), generator=gen, device="cuda") + 0.5
    _, _, mean, rstd = training.layer_norm(x, w, b)
    _, dw, db = training.layer_norm_grad(d, x, mean, rstd, w, b)
    sums = torch.zeros((2, C), dtype=torch.float64, device="cuda")
    step = 100_000_000 // C
    for i in range(0, N, step):
        at = slice(i, i + step)
        xh = (x[at].double() - mean[at].double()[:, None]) * rstd[at].double()[:, None]
        sums += torch.stack([d[at].double().sum(0), (d[at].double() * xh).sum(0)])
    for got, want in ((db, sums[0]), (dw, sums[1])):
        assert float((got.double() - want).norm() / want.norm()) <= (run / 6 + 5 / 3) ** 0.5 * 2.0**-24
