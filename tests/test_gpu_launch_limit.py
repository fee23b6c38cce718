"""Launches of 2^32 threads or more, which HIP would cut to the remainder
without an error: the library refuses them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_pack_of_more_threads_than_a_launch_has(gpu):
    """64 threads a row of 256 features, over 2^26 rows (69 GB, any values)."""
    from tcc_amd import _lib, swtcf

    x = torch.empty((2**26 + 8, 256), device="cuda")
    with pytest.raises(_lib.TccError):
        swtcf.tf32_pack(x)
    assert swtcf.tf32_pack(x[:64].zero_()).numel() > 0  # and the error is gone
