"""tvk_rms_norm_fwd / tvk_rms_norm_bwd against the formulas in float64.

Tolerances count roundings. u = 2^-24 is half a float32 step; a row's float32
sums over c columns go through at most c / 256 + 8 additions in any one chain,
and a handful of products, a square root and a division follow: everything
before the last rounding is off by at most f = 2 (c / 256 + 32) u of the sum
of its terms' magnitudes. The output's rounding adds half a step of its type
(eps / 2 of the value, or half the smallest subnormal)."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from torchvulkan_amd import _abi

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def rand(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def half_step(t, dtype):
    return torch.finfo(dtype).eps / 2 * t.abs() + TINY[dtype]


def oracle(x, w, r, eps):
    """(h, y) on the CPU: h in x's dtype, y in float64."""
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    d = h.double()
    y = d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    return h, y if w is None else y * w.double()


def oracle_bwd(dy, h, w, dh, eps):
    """(dx, dw, dx's magnitude, dw's magnitude) in float64."""
    h, g = h.double(), dy.double() if w is None else dy.double() * w.double()
    inv = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    n = h * inv
    dx = inv * (g - n * (g * n).mean(-1, keepdim=True))
    size = inv * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    if dh is not None:
        dx, size = dx + dh.double(), size + dh.double().abs()
    return dx, (dy.double() * n).sum(0), size, (dy.double() * n).abs().sum(0)


def factor(cols):
    return 2 * (cols / 256 + 32) * U


def close(got, ref, tol, what):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), f"{what}: NaN in other places"
    over = ((got - ref).abs() - tol).nan_to_num(nan=-1.0)
    assert over.max() <= 0, f"{what}: {over.max().item():.3e} over the tolerance"


def check_fwd(x, w=None, r=None, eps=1e-5, out8=False, what=""):
    h, y = oracle(x, w, r, eps)
    dev = [None if t is None else t.to(DEV) for t in (x, w, r)]
    got, got_h, scale = _abi.rms_norm_fwd(dev[0], dev[1], dev[2], eps, torch.float8_e4m3fn if out8 else None)
    torch.cuda.synchronize()
    close(got_h, h.double(), torch.zeros_like(h.double()), what + " h")
    f = factor(x.shape[1])
    if not out8:
        close(got, y, f * y.abs() + half_step(y, x.dtype), what)
        return
    top = y.abs().amax(-1)
    s = torch.where(top > 0, top / 448, 1.0)
    close(scale, s, 2 * f * s + TINY[torch.float32], what + " scale")
    t = y / s[:, None]
    close(got.float(), t, (2.0 ** -4 + 4 * f) * t.abs() + 2.0 ** -10, what + " 8 bits")


def check_bwd(dy, h, w=None, dh=None, eps=1e-5, what=""):
    dx, dw, size, wsize = oracle_bwd(dy, h, w, dh, eps)
    dev = [None if t is None else t.to(DEV) for t in (dy, h, w, dh)]
    got, got_w = _abi.rms_norm_bwd(*dev, eps=eps)
    torch.cuda.synchronize()
    f = factor(h.shape[1])
    close(got, dx, f * size + half_step(dx, h.dtype), what + " dx")
    if w is not None:
        close(got_w, dw, (f + h.shape[0] * U) * wsize + half_step(dw, w.dtype), what + " dw")


# one column, below and at a wave, odd, the sizes where a row's share of a thread changes, past the widest of them
COLS = [1, 7, 64, 100, 128, 511, 512, 777, 1024, 2047, 2048, 2056, 4096, 8191, 8192, 16384, 20001]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward(gpu, cols, dtype):
    x, w, r = rand((5, cols), dtype, cols), rand((cols,), dtype, 1) + 1, rand((5, cols), dtype, 2, 3.0)
    check_fwd(x, w, r, what=f"{cols} {dtype}")
    check_fwd(x, w.float(), what=f"{cols} {dtype} float32 weight")
    check_fwd(x, what=f"{cols} {dtype} no weight")
    check_fwd(x, w, r, out8=True, what=f"{cols} {dtype}")


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_backward(gpu, cols, dtype):
    dy, h, w, dh = rand((9, cols), dtype, cols), rand((9, cols), dtype, 1, 2.0), rand((cols,), dtype, 2), rand((9, cols), dtype, 3)
    check_bwd(dy, h, w, dh, what=f"{cols} {dtype}")
    check_bwd(dy, h, w.float(), what=f"{cols} {dtype} float32 weight")
    check_bwd(dy, h, None, dh, what=f"{cols} {dtype} no weight")


@pytest.mark.parametrize("rows,cols", [(1, 4096), (2, 96), (255, 1000), (1025, 520), (5000, 128), (3001, 64), (70000, 8)])
def test_rows(gpu, rows, cols):
    dtype = torch.bfloat16 if rows % 2 else torch.float16
    x, w = rand((rows, cols), dtype, 1), rand((cols,), dtype, 2)
    check_fwd(x, w, rand((rows, cols), dtype, 3), what=f"{rows}x{cols}")
    check_fwd(x, w, out8=True, what=f"{rows}x{cols}")
    check_bwd(rand((rows, cols), dtype, 4), x, w, what=f"{rows}x{cols}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_values(gpu, dtype):
    # zero rows (with and without eps they stay finite only by eps), tiny and large ones, infinities and NaN
    x = rand((8, 200), dtype, 1)
    x[0] = 0
    x[1] *= 2.0 ** -14
    x[2] *= 100
    x[3, 5] = float("inf")
    x[4, 6] = float("nan")
    x[5, :] = 0
    x[5, 9] = 1
    w = rand((200,), dtype, 2)
    check_fwd(x, w, what="values")
    h, y = oracle(x, w, None, 1e-5)
    got, _, scale = _abi.rms_norm_fwd(x.to(DEV), w.to(DEV), out_dtype=torch.float8_e4m3fn)
    got, scale = got.float().cpu(), scale.cpu()
    assert got[0].eq(0).all() and scale[0] == 1
    assert got[3, 5].isnan() and got[3, :5].eq(0).all()
    assert got[4].isnan().all()


def test_zero_rows_without_eps(gpu):
    # 0 / 0: NaN, as the formula has it
    x = torch.zeros((2, 64), dtype=torch.float16)
    got, _, _ = _abi.rms_norm_fwd(x.to(DEV), eps=0.0)
    assert got.isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [96, 2048, 20001])
def test_strides_and_places(gpu, dtype, cols):
    # rows inside wider ones and at odd offsets, results over their inputs
    wide = rand((6, cols + 13), dtype, 1)
    w = rand((cols + 1,), dtype, 2)[1:]
    r = rand((6, 2 * cols), dtype, 3)[:, ::2].contiguous()
    h, y = oracle(wide[:, 3:3 + cols], w, r, 1e-5)
    f = factor(cols)
    x = wide.to(DEV)[:, 3:3 + cols]
    wd, rd = w.to(DEV), r.to(DEV)
    wd = torch.cat([wd[:1], wd])[1:]
    out = torch.full((6, cols + 5), 7.0, dtype=dtype, device=DEV)
    lib = _abi.load()
    d = _abi.make_rms_norm_desc(x, wd, out[:, 1:1 + cols], residual=rd, residual_out=rd,
                                stream=torch.cuda.current_stream().cuda_stream)
    _abi.check(lib.tvk_rms_norm_fwd(C.byref(d)))
    assert torch.equal(rd.cpu(), h)
    close(out[:, 1:1 + cols], y, f * y.abs() + half_step(y, dtype), "strides")
    assert out[:, 0].eq(7).all() and out[:, 1 + cols:].eq(7).all()
    # the output over x
    xd = wide.to(DEV)
    d = _abi.make_rms_norm_desc(xd[:, 3:3 + cols], wd, xd[:, 3:3 + cols], residual=r.to(DEV), residual_out=rd,
                                stream=torch.cuda.current_stream().cuda_stream)
    _abi.check(lib.tvk_rms_norm_fwd(C.byref(d)))
    close(xd[:, 3:3 + cols], y, f * y.abs() + half_step(y, dtype), "over x")
    assert torch.equal(xd[:, :3].cpu(), wide[:, :3]) and torch.equal(xd[:, 3 + cols:].cpu(), wide[:, 3 + cols:])
    # dx over dy, over h, over dh
    dy, dh = rand((6, cols), dtype, 4), rand((6, cols), dtype, 5)
    dx, dw, size, wsize = oracle_bwd(dy, h, w, dh, 1e-5)
    for over in range(3):
        t = [dy.to(DEV), h.to(DEV), dh.to(DEV)]
        gw = torch.empty_like(wd)
        d = _abi.make_rms_norm_bwd_desc(t[0], t[1], wd, t[over], gw, dh=t[2],
                                        stream=torch.cuda.current_stream().cuda_stream)
        _abi.check(lib.tvk_rms_norm_bwd(C.byref(d)))
        close(t[over], dx, f * size + half_step(dx, dtype), f"dx over {over}")
        close(gw, dw, (f + 6 * U) * wsize + half_step(dw, dtype), f"dw over {over}")


def test_no_rows(gpu):
    w = rand((64,), torch.float16, 1).to(DEV)
    x = torch.empty((0, 64), dtype=torch.float16, device=DEV)
    y, _, _ = _abi.rms_norm_fwd(x, w)
    dx, dw = _abi.rms_norm_bwd(x, x, w)
    assert y.shape == dx.shape == (0, 64) and dw.eq(0).all()


@pytest.mark.parametrize("rows,cols", [(3000, 512), (300, 4096), (40, 20001)])
def test_same_bits(gpu, rows, cols):
    dy, h, w = (rand(s, torch.bfloat16, i).to(DEV) for i, s in enumerate([(rows, cols), (rows, cols), (cols,)]))
    first = _abi.rms_norm_bwd(dy, h, w)
    for _ in range(3):
        again = _abi.rms_norm_bwd(dy, h, w)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_streams_and_capture(gpu):
    rows, cols = 2000, 1024
    dy, h, w = (rand(s, torch.float16, i).to(DEV) for i, s in enumerate([(rows, cols), (rows, cols), (cols,)]))
    dx, dw = torch.empty_like(h), torch.empty_like(w)
    y = torch.empty((rows, cols), dtype=torch.float8_e4m3fn, device=DEV)
    scale = torch.empty(rows, device=DEV)
    lib = _abi.load()

    def calls(stream):
        f = _abi.make_rms_norm_desc(h, w, y, scale=scale, stream=stream)
        b = _abi.make_rms_norm_bwd_desc(dy, h, w, dx, dw, stream=stream)
        _abi.check(lib.tvk_rms_norm_fwd(C.byref(f)))
        _abi.check(lib.tvk_rms_norm_bwd(C.byref(b)))

    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        calls(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        h.copy_(rand((rows, cols), torch.float16, 10 + i))
        torch.cuda.synchronize()
        want = _abi.rms_norm_fwd(h, w, out_dtype=torch.float8_e4m3fn), _abi.rms_norm_bwd(dy, h, w)
        for t in (dx, dw, scale):
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.view(torch.uint8), want[0][0].view(torch.uint8)) and torch.equal(scale, want[0][2])
        assert torch.equal(dx, want[1][0]) and torch.equal(dw, want[1][1])


# more rows than a launch has workgroups to give one each: a wave, a part of one or several to a row, with rows left over
@pytest.mark.parametrize("cols", [96, 129, 250, 513, 640, 1023, 1024, 2050, 4099])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(gpu, cols, dtype):
    rows = 2051
    x, w, r = rand((rows, cols), dtype, cols), rand((cols,), dtype, 1) + 1, rand((rows, cols), dtype, 2, 3.0)
    check_fwd(x, w, r, what=f"{cols} {dtype}")
    check_fwd(x, w.float(), out8=True, what=f"{cols} {dtype} 8 bits, float32 weight")
    check_bwd(r, x, w, rand((rows, cols), dtype, 3), what=f"{cols} {dtype}")
    check_bwd(r, x, w.float(), what=f"{cols} {dtype} float32 weight")


@pytest.mark.parametrize("cols", [200, 1500])
def test_many_rows_in_place(gpu, cols):
    # rows inside wider ones at odd offsets, the output over x, dx over dh, inputs shared by all rows
    rows, dtype = 2051, torch.float16
    wide = rand((rows, cols + 3), dtype, 1)
    w, one = rand((cols,), dtype, 2), rand((1, cols), dtype, 3).expand(rows, cols)
    h, y = oracle(wide[:, 1:1 + cols], w, one, 1e-5)
    xd, od = wide.to(DEV), one[:1].to(DEV).expand(rows, cols)
    lib, stream = _abi.load(), torch.cuda.current_stream().cuda_stream
    wd, hd = w.to(DEV), torch.empty((rows, cols), dtype=dtype, device=DEV)
    d = _abi.make_rms_norm_desc(xd[:, 1:1 + cols], wd, xd[:, 1:1 + cols], residual=od, residual_out=hd, stream=stream)
    _abi.check(lib.tvk_rms_norm_fwd(C.byref(d)))
    f = factor(cols)
    assert torch.equal(hd.cpu(), h)
    close(xd[:, 1:1 + cols], y, f * y.abs() + half_step(y, dtype), "over x")
    assert torch.equal(xd[:, 0].cpu(), wide[:, 0]) and torch.equal(xd[:, 1 + cols:].cpu(), wide[:, 1 + cols:])
    dh = rand((rows, cols), dtype, 5)
    dx, dw, size, wsize = oracle_bwd(one, h, w, dh, 1e-5)
    t, gw = dh.to(DEV), torch.empty_like(wd)
    d = _abi.make_rms_norm_bwd_desc(od, hd, wd, t, gw, dh=t, stream=stream)
    _abi.check(lib.tvk_rms_norm_bwd(C.byref(d)))
    close(t, dx, f * size + half_step(dx, dtype), "dx over dh")
    close(gw, dw, (f + rows * U) * wsize + half_step(dw, dtype), "dw")


@pytest.mark.parametrize("cols", [64, 300, 2048])
def test_8bit_rows_near_the_ends_of_float32(gpu, cols):
    # scales beside which one over the other leaves float32: tiny rows without eps, large ones
    x = rand((3, cols), torch.float32, 1)
    x[0] *= 2.0 ** -50
    x[1] *= 2.0 ** 50
    w = torch.ones(cols) * 2.0 ** -80
    check_fwd(x, w, eps=0.0, out8=True, what="tiny weights")
    check_fwd(x, w * 2.0 ** 140, eps=0.0, out8=True, what="large weights")
