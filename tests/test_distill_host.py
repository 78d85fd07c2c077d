"""Refusals of the distillation loss that need no GPU: every call fails before any launch."""
import pytest

import unet_amd
from unet_amd import _lib


@pytest.mark.parametrize("weight,temperature", [(1e39, 1.0), (1e30, 1e6), (-1e38, 1e2)])
def test_scales_beyond_fp32_are_refused(weight, temperature):
    """weight * temperature**2 scales the loss: infinite, it would make NaN of a row whose divergence is 0."""
    with pytest.raises(ValueError, match="fp32"):
        unet_amd.TopLogitDistillationLoss(temperature, weight=weight)
    unet_amd.TopLogitDistillationLoss(temperature, weight=weight * 1e-12)


def test_scales_beyond_fp32_are_refused_at_the_c_entry():
    lib = _lib.load()

    def fwd(temperature, weight):
        return lib.mi_distill_loss_fwd(1, 4, 16, 16, 4096, 4, 0, 4096, 3, 4096, temperature, weight, 1, 4096, 4096, None)

    assert fwd(1e6, 1e30) != 0 and b"temperature^2" in lib.mi_last_error()
    assert fwd(1.0, float("inf")) != 0 and b"finite" in lib.mi_last_error()
