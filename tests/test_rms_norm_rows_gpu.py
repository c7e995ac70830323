"""Rows without values, and their scales in 8 bits."""
import pytest
import torch

from torchvulkan_amd import _abi, decoder

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("device", ["cuda", "vulkan"])
@pytest.mark.parametrize("shape", [(3, 5, 0), (0, 0), (0, 8), (0,), (100000, 0)])
def test_rows_without_values(gpu, device, shape):
    x = torch.zeros(shape, dtype=torch.bfloat16).to(device)
    y, h = decoder.rms_norm(x, None, x)
    assert y.shape == h.shape == x.shape
    torch.full((x.numel() + 100000,), 7.0).to(device)   # what an allocation that is not written may hold
    y, scale, h = decoder.rms_norm_fp8(x)
    assert y.shape == h.shape == x.shape and scale.shape == x.shape[:-1]
    assert scale.cpu().eq(1).all()   # no value, so all zero
    _, dw = _abi.rms_norm_bwd(*(torch.zeros((3, 0), device="cuda") for _ in range(2)), torch.zeros(0, device="cuda"))
    assert dw.shape == (0,)
