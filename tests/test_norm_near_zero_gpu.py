"""Values that a layer norm takes to nearly zero, of rows whose mean is a small part of their deviation.

Such a value's distance d from the mean is a float32 that is off by 2^-24 of itself and by the mean's own rounding, which is the
mean of many additions'. An addition whose result is p is off by at most u |p| / sqrt(3) root mean square, u = 2^-24. Over a
row of 4096 float32 values of deviation s in 1024 threads, with sums of k values being about sqrt(k) s: 9 s^2 a thread (2 + 3 + 4
values), 4096 s^2 at each of 6 steps between lanes, (2 + .. + 16) 256 s^2 over 16 waves; in all 68000 s^2, and so 151 u s of
the row's sum and 0.037 u s of its mean; the product with 1 / 4096 leaves u / sqrt(3) of the mean itself, s / 64 on the whole,
0.01 u s. So values within s / 1000 of the mean come out within 0.04 u root mean square, and within as much again for other
shapes' sums: 0.1 u is allowed. (Their own roundings are 14 u / 1000 at most.)

Rows past what registers hold are added by 256 threads, cols / 256 values each one after the other. The values here are of few
bits, the row's own small number aside, so that the k-th additions of all threads have the same bits to round off and their
errors do not average: with a = u sqrt(k) s / sqrt(3) for the k-th, 256 sqrt(sum of a^2) = 256 u s sqrt(12250 / 3) = 16400 u s of the
row's sum for 40000 columns, which is 0.41 u s of its mean: 0.5 u is allowed there."""
from __future__ import annotations

import pytest
import torch

from torchvulkan_amd import _abi

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
ROWS = 1024


def allowed(cols):
    return (0.1 if cols <= 16384 else 0.5) * U


def rows_and_norm(cols, seed):
    """Rows of values that bfloat16 holds, in float32, and their norms in 64 bits."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn((ROWS, cols), generator=g, device=DEV) * 2).bfloat16().float()
    x += (torch.rand((ROWS, 1), generator=g, device=DEV) * 0.03).bfloat16().float()
    d = x.double() - x.double().mean(-1, keepdim=True)
    return x, d / (d * d).mean(-1, keepdim=True).add(1e-5).sqrt()


@pytest.mark.parametrize("cols", [1024, 4096, 8192, 40000])
def test_forward(gpu, cols):
    x, n = rows_and_norm(cols, cols)
    y, _, _ = _abi.layer_norm_fwd(x)
    near = n.abs() < 1e-3
    assert near.sum() > 500
    assert (y.double() - n)[near].pow(2).mean().sqrt().item() <= allowed(cols)


@pytest.mark.parametrize("cols", [1024, 4096, 8192, 40000])
def test_backward(gpu, cols):
    """dweight of a column is n at the row that has the column's only dy."""
    x, n = rows_and_norm(cols, cols + 1)
    at = n.abs().argmin(0)
    dy = torch.zeros_like(x)
    dy[at, torch.arange(cols, device=DEV)] = 1
    _, dweight, _ = _abi.layer_norm_bwd(dy, x)
    want = n[at, torch.arange(cols, device=DEV)]
    near = want.abs() < 1e-3
    assert near.sum() > 500
    assert (dweight.double() - want)[near].pow(2).mean().sqrt().item() <= allowed(cols)


def test_between(gpu):
    """Means from a hundredth of the deviation to a hundred times it: values near the mean are off by the roundings of d or
    by the mean's. Either is a few u: d's are u |d| each, u on the whole, the mean's up to u |mean| sqrt(20 / 3) where it is not
    taken off, for |mean| < s / 8."""
    for mean in (0.02, 0.1, 0.24, 0.26, 0.5, 2.0, 20.0, 200.0):
        x, _ = rows_and_norm(4096, 5)
        x = x + torch.tensor(mean)
        d = x.double() - x.double().mean(-1, keepdim=True)
        n = d / (d * d).mean(-1, keepdim=True).add(1e-5).sqrt()
        y, _, _ = _abi.layer_norm_fwd(x)
        near = n.abs() < 1e-3
        assert (y.double() - n)[near].pow(2).mean().sqrt().item() <= 2 * U, mean
