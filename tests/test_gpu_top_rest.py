"""The rest of tcc_amd.training.top_logits where it has no finite value."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BY_DTYPE = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])


@pytest.mark.parametrize("C", [6, 12, 70, 500, 900, 3000, 6000])
@BY_DTYPE
def test_rest_of_an_infinity_and_a_nan(gpu, dtype, C):
    """log(exp(inf) + NaN) is NaN, log(exp(inf)) infinite, whatever else there is."""
    from tcc_amd import training

    gen = torch.Generator().manual_seed(C)
    n = 8 if C < 6000 else 12 * torch.cuda.get_device_properties(0).multi_processor_count
    z = torch.randn((n, C), generator=gen).to(dtype)
    z[0, 1:4], z[0, 5] = np.nan, np.inf
    z[1, [0, 2, C - 1]], z[1, 3] = np.nan, np.inf
    z[2, 1:3], z[2, 4] = np.nan, np.inf
    z[3, :4] = np.inf
    z[4, 2], z[4, 3:5] = np.nan, np.inf
    z[5, :4], z[5, 4:] = np.nan, np.inf
    z[6, 0], z[6, 4:], z[6, 1:4] = np.nan, -np.inf, np.inf
    z = z.cuda()
    _, _, rest = training.top_logits(z, 2, temperature=3.0)
    assert bool(rest[[0, 1, 5]].isnan().all())
    assert bool((rest[[2, 3, 4, 6]] == np.inf).all())
    assert bool(torch.isfinite(rest[7]).all())
