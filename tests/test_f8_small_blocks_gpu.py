"""8-bit blocks whose values are next to nothing: finite values stay finite, within half a step of an 8-bit number times
the block's scale.

A step of e4m3 at v is 2^-3 of the power of two at or below |v|, and 2^-9 below 2^-6. So with the stored scale s, in 64 bits,
|q s - x| is at most 2^-4 |x| and at most 2^-10 s where the value is a subnormal number; the quotient's rounding on the way
(2^-23 of it at most) may take a value on the border to the other neighbour, which is 2^-23 |x| farther away. The largest of a
block may be past 448 by the scale's own rounding, 2^-7 of it at most: it becomes 448, within 2^-4 of it too."""
from __future__ import annotations

import math

import pytest
import torch

from torchvulkan_amd import _abi, decoder

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
F8 = torch.float8_e4m3fn
TOPS = [1.4e-45, 3e-44, 3.1e-43, 3.2e-43, 4e-42, 9e-42, 1e-41, 4e-41, 1e-39, 1e-37, 1e-30]


def rows_of(top, rows, cols, seed):
    """Values up to `top`, which is among them, and zeros."""
    x = torch.rand((rows, cols), generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * 2 - 1
    x[:, ::7] = 0
    x[:, 3::128] = 1
    return (x * top).float()


def check_values(x, q, scale, tall=1):
    x, q = x.double().cpu(), q.cpu().float().double()
    s = scale.cpu().double().repeat_interleave(tall, 0)[:x.shape[0]].repeat_interleave(128, 1)[:, :x.shape[1]]
    assert q.isfinite().all() and s.isfinite().all() and (s > 0).all()
    off = (q * s - x).abs() - x.abs() * (2.0 ** -4 + 2.0 ** -22) - s * 2.0 ** -10
    assert off.max() <= 0
    assert not q[x == 0].any()


@pytest.mark.parametrize("top", TOPS)
def test_quantize(gpu, top):
    x = rows_of(top, 130, 300, 1)
    for tall in (1, 128):
        q, scale = _abi.quantize_f8(x.to(DEV), tall)
        check_values(x, q, scale, tall)


def test_ends_of_the_range(gpu):
    """Large values, small ones and those that are none, in blocks of their own."""
    x = torch.randn((6, 256), generator=torch.Generator().manual_seed(0))
    x[0] *= 1e38 / 4
    x[1] *= 1e-38
    x[2] *= 1e-44
    x[3, 7], x[4, 9], x[4, 200] = math.nan, math.inf, -math.nan
    q, s = _abi.quantize_f8(x.to(DEV))
    plain = torch.ones(x.shape, dtype=torch.bool)
    plain[3, 7] = plain[4] = False
    top = x.abs().nan_to_num(nan=0.0).view(6, 2, 128).amax(-1)
    assert torch.equal(s.cpu()[[0, 1, 3, 5]], (top / 448)[[0, 1, 3, 5]])
    check_values(torch.where(plain, x, 0.0)[[0, 1, 2, 5]], q[[0, 1, 2, 5]], s[[0, 1, 2, 5]])
    got = q.cpu().float()
    assert got[3, 7].isnan() and got[3].isnan().sum() == 1
    assert got[4, 9].isnan() and not got[4, :9].any() and got[4, 200].isnan() and got[4, 128:].isnan().sum() == 1


@pytest.mark.parametrize("top", TOPS)
@pytest.mark.parametrize("cols", [300, 4096, 17000, 40000])
def test_layer_norm(gpu, top, cols):
    """Through the gains: each form of the kernel."""
    x = torch.randn((3, cols), generator=torch.Generator().manual_seed(2))
    w = torch.full((cols,), top)
    y, _, _ = _abi.layer_norm_fwd(x.to(DEV), w.to(DEV))
    q, _, scale = _abi.layer_norm_fwd(x.to(DEV), w.to(DEV), out_dtype=F8)
    check_values(y, q, scale)


@pytest.mark.parametrize("m", [1, 5, 20, 100])
def test_product(gpu, m):
    """One block of a row, and one of the weight, next to nothing: finite rows and columns, as near the product in 64 bits
    as the 8 bits allow (2^-4 of either factor and 2^-10 of its block's largest / 448, beside float32's 2^-13 of all). A block's
    sum of codes' products goes times its two scales' product, which is a multiple of 2^-149 where it is below float32's normal
    range, and so off by 2^-150 at most: 2^-150 of the codes' products is allowed, and 2^-150 for each block's addition."""
    k, n = 300, 260
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(3))
    w = torch.randn((n, k), generator=torch.Generator().manual_seed(4))
    for row, top in enumerate((3e-44, 4e-42, 1e-41)[:m]):
        x[row, 128:256] = rows_of(top, 1, 128, row)[0]
    x[0, :128] = x[0, 256:] = 0
    w[128:256, :128] = rows_of(4e-42, 128, 128, 9)
    q, scale = _abi.quantize_f8(w.to(DEV), 128)
    for a, a_scale in ((x.to(DEV), None), _abi.quantize_f8(x.to(DEV))):
        got = _abi.gemm_f8(a, a_scale, q, scale, out_dtype=torch.float32).cpu().double()
        xd, wd = x.double(), w.double()
        dx, dw = xd.abs() * 2.0 ** -4 + xd.abs().amax() / 448 * 2.0 ** -10, wd.abs() * 2.0 ** -4 + wd.abs().amax() / 448 * 2.0 ** -10
        tol = (xd.abs() + dx) @ dw.t() + dx @ wd.abs().t() + 2.0 ** -13 * (xd.abs() @ wd.abs().t())
        codes = _abi.quantize_f8(x.to(DEV))[0].cpu().float().double().abs() @ q.cpu().float().double().abs().t()
        tol = tol * 1.01 + 2.0 ** -150 * (codes + 4)
        assert bool(got.isfinite().all()) and bool(((got - xd @ wd.t()).abs() <= tol).all())


def test_entry_points(gpu):
    x = rows_of(4e-42, 9, 300, 5).to(DEV)
    q, scale = decoder.quantize_fp8(x)
    check_values(x, q, scale)
    out = decoder.linear_fp8(x, *decoder.quantize_fp8(torch.ones((40, 300), device=DEV) * 1e30, 128))
    ref = x.double().cpu().sum(-1) * 1e30
    size = x.double().cpu().abs().sum(-1) * 1e30
    assert ((out.double().cpu() - ref[:, None]).abs() <= (size * 0.07)[:, None]).all()
