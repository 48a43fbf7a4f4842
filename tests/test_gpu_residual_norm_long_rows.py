"""The norms around a block on long rows of odd lengths, several of them to a
work-group, with and without biases and shared gates, against 64 bits."""
import pytest
import torch

from test_gpu_residual_norm import TYPES, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [4099, 7195, 8191, 8193, 12289])
@pytest.mark.parametrize("affine", [0, 1])
def test_odd_long_rows(dtype, channels, affine):
    _check(3, channels, dtype, "RMS", "LAYER", "NONE", 1, affine=affine)
    _check(600, channels, dtype, "LAYER", "RMS", "SILU", 251, affine=affine)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_long_rows(dtype):
    _check(2500, 5000, dtype, "RMS", "RMS", "VALUE", 1)
