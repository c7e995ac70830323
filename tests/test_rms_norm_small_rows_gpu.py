"""8-bit rows of the root-mean-square norm whose values are next to nothing: finite values stay finite, within half a step
of an 8-bit number times the row's scale (2^-4 of the value, 2^-10 of the scale), beside the roundings on the way: h w and
its product with 1 / sqrt(mean), multiples of 2^-149 each, so 2^-148 here, and 2^-20 of the value."""
from __future__ import annotations

import pytest
import torch

from torchvulkan_amd import _abi, decoder

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
F8 = torch.float8_e4m3fn


@pytest.mark.parametrize("top", [1.4e-45, 3e-44, 3.1e-43, 4e-42, 9e-42, 1e-41, 1e-39, 1e-37])
@pytest.mark.parametrize("cols", [130, 1000, 4099, 40000])
def test_finite_rows(gpu, cols, top):
    x = torch.randn((3, cols), generator=torch.Generator().manual_seed(cols))
    x[:, ::5] = 0
    w = torch.full((cols,), top)
    q, _, scale = _abi.rms_norm_fwd(x.to(DEV), w.to(DEV), out_dtype=F8)
    y = x.double() / (x.double() ** 2).mean(-1, keepdim=True).add(1e-5).sqrt() * w.double()
    q, s = q.cpu().float().double(), scale.cpu().double()[:, None]
    assert bool(q.isfinite().all()) and bool((s > 0).all()) and not bool(q[:, ::5].any())
    off = (q * s - y).abs() - (2.0 ** -4 + 2.0 ** -20) * y.abs() - 2.0 ** -10 * s - 2.0 ** -148
    assert off.max().item() <= 0
    q2, scale2, _ = decoder.rms_norm_fp8(x.to(DEV), w.to(DEV))
    assert torch.equal(q2.cpu().view(torch.uint8), q.float().to(F8).view(torch.uint8)) and torch.equal(scale2, scale)
