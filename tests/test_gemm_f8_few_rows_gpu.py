"""8-bit products of up to 4 rows in wider types on both sides of the column counts at which workgroups take more of W: the
bits of the rows brought into 8 bits beforehand, whose sums run in the same order."""
from __future__ import annotations

import pytest
import torch

from torchvulkan_amd import _abi

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.mark.parametrize("n", [8192, 8193, 12288, 12289, 16384, 16385])
@pytest.mark.parametrize("k", [640, 1100])
def test_either_side(gpu, n, k):
    g = torch.Generator(device=DEV).manual_seed(n)
    w, w_scale = _abi.quantize_f8(torch.randn((n, k), generator=g, device=DEV), 128)
    for m in (1, 3, 4, 5):
        for dtype in (torch.float32, torch.float16, torch.bfloat16):
            x = torch.randn((m, k), generator=g, device=DEV).to(dtype)
            q, scale = _abi.quantize_f8(x)
            want = _abi.gemm_f8(q, scale, w, w_scale, out_dtype=dtype)
            assert torch.equal(_abi.gemm_f8(x, None, w, w_scale), want)
            ref = (q.float() * scale.repeat_interleave(128, 1)[:, :k]).double() @ \
                (w.float() * w_scale.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]).double().t().contiguous()
            # sums of 8-bit products cut off 2^-13 below the largest of eight, and the result's rounding
            assert ((want.double() - ref).abs() <= ref.abs() * torch.finfo(dtype).eps + 2.0 ** -9 * ref.abs().amax()).all()
