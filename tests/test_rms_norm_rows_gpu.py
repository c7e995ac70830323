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


@pytest.mark.parametrize("cols", [8193, 10007])
def test_long_rows_by_workgroups_in_turn(gpu, cols):
    # more rows than the launch has workgroups; rows are views of one vector, each a value further on
    rows, dev = (1 << 16) + 3, "cuda"
    g = torch.Generator(device=dev).manual_seed(cols)
    base, base2 = (torch.randn(rows + cols, generator=g, device=dev) for _ in range(2))
    x, dy = base.as_strided((rows, cols), (1, 1)), base2.as_strided((rows, cols), (1, 1))
    w = torch.randn(cols, generator=g, device=dev)
    u, eps = 2.0 ** -24, 1e-5
    y, _, _ = _abi.rms_norm_fwd(x, w, eps=eps)
    y8, _, scale = _abi.rms_norm_fwd(x, w, eps=eps, out_dtype=torch.float8_e4m3fn)
    dx, dw = _abi.rms_norm_bwd(dy, x, w, eps=eps)
    want_dw, size_dw = torch.zeros(cols, dtype=torch.float64, device=dev), torch.zeros(cols, dtype=torch.float64, device=dev)
    for r in range(0, rows, 4096):
        h, d, wd = x[r:r + 4096].double(), dy[r:r + 4096].double(), w.double()
        inv = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
        n, gr = h * inv, d * wd
        # the sum of squares is off by its number of terms a thread and the workgroup's; half of that in its root, and the product
        tol = (cols / 256 + 64) * u
        assert ((y[r:r + 4096].double() - n * wd).abs() <= tol * (n * wd).abs()).all()
        got8 = y8[r:r + 4096].double() * scale[r:r + 4096, None].double()
        assert ((got8 - n * wd).abs() <= (2.0 ** -4 + tol) * (n * wd).abs() + 2.0 ** -10 * scale[r:r + 4096, None].double()).all()
        mean, size = (gr * n).mean(-1, keepdim=True), (gr * n).abs().mean(-1, keepdim=True)
        want = inv * (gr - n * mean)
        assert ((dx[r:r + 4096].double() - want).abs() <= 3 * tol * inv * (gr.abs() + n.abs() * size)).all()
        want_dw += (d * n).sum(0)
        size_dw += (d * n).abs().sum(0)
    # a thread adds every 256th row, then 4 waves and 64 partials
    assert ((dw.double() - want_dw).abs() <= (rows / 256 + 4 + 64 + cols / 256 + 64) * u * size_dw).all()
