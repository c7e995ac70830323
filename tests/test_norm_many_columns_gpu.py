"""Gradients of norms of so many columns that a grid in a line would have 2^32 threads or more."""
from __future__ import annotations

import pytest
import torch

from torchvulkan_amd import _abi

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_gradients_of_many_columns(gpu, kind):
    """2^26 columns and three more, one row: dweight is dy n. The row's sums go through cols / 256 + 8 additions in a chain: each
    is off by at most f = (cols / 256 + 32) u of its terms' magnitudes, and n by f of itself and of 1 at most (the mean's, of
    mean|x|); bfloat16's rounding adds 2^-9 of the value."""
    cols = (1 << 26) + 3
    g = torch.Generator(device=DEV).manual_seed(1)
    h, dy = (torch.randn((1, cols), generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    weight = torch.ones(cols, device=DEV, dtype=torch.bfloat16)
    if kind == "layer":
        _, dweight, dbias = _abi.layer_norm_bwd(dy, h, weight)
        assert torch.equal(dbias, dy[0])
    else:
        dweight = _abi.rms_norm_bwd(dy, h, weight)[1]
    f = (cols / 256 + 32) * 2.0 ** -24
    x = h[0].double()
    if kind == "layer":
        x -= x.mean()
    x /= (x * x).mean().add(1e-5).sqrt()
    want = x * dy[0].double()
    tol = dy[0].double().abs() * f * (x.abs() + 1) + want.abs() * 2.0 ** -8 + 2.0 ** -134
    assert ((dweight.double() - want).abs() <= tol).all()
