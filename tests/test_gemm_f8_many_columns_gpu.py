"""8-bit products of so many columns that a grid in a line would have 2^32 threads or more."""
from __future__ import annotations

import pytest
import torch

from torchvulkan_amd import _abi

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
F8 = torch.float8_e4m3fn


@pytest.mark.parametrize("m,dtype", [(1, F8), (3, torch.bfloat16)])
def test_product_of_many_columns(gpu, m, dtype):
    """2^27 rows of W and five more, one row for all of them; the results differ by their biases."""
    n, k = (1 << 27) + 5, 16
    w, one = torch.full((1, k), 0.25, device=DEV).to(F8).expand(n, k), torch.ones((1, 1), device=DEV)
    bias = (torch.arange(n, device=DEV, dtype=torch.int32) % 251).to(torch.bfloat16)
    a = torch.ones((m, k), device=DEV).to(dtype)
    out = _abi.gemm_f8(a, one.expand(m, 1) if dtype == F8 else None, w, one.expand(-(-n // 128), 1), bias, torch.bfloat16)
    bias += 4
    assert all(torch.equal(row, bias) for row in out)
