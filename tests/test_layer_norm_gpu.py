"""tvk_layer_norm_fwd / tvk_layer_norm_bwd against the formulas in float64.

Tolerances count roundings. u = 2^-24 is half a float32 step; a row's float32
sums over c columns go through at most c / 256 + 8 additions in any one chain,
and a handful of products, a square root and a division follow: every sum is off
by at most f = 2 (c / 256 + 32) u of the sum of its terms' magnitudes. The mean
m that the first sum gives is off by f mean|x|; the centred values take that off
again as e, which is off by f mean|d| and by the rounding u of d = x - m, where
|d| <= |x - mean| + f mean|x|. So with n = (x - mean) inv a centred value times
inv is off by at most 2 f (|n| + 1 + f mean|x| inv), and the variance, two sums
of squares whose difference it is, by f (1 + (f mean|x| inv)^2) of itself. The
output's rounding adds half a step of its type (eps / 2 of the value, or half the
smallest subnormal)."""
from __future__ import annotations

import pytest
import torch

from torchvulkan_amd import _abi, decoder

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def rand(shape, dtype, seed, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std + mean).to(dtype)


def half_step(t, dtype):
    return torch.finfo(dtype).eps / 2 * t.abs() + TINY[dtype]


def factor(cols):
    return 2 * (cols / 256 + 32) * U


def stats(h, eps):
    """(n, inv, n's error) of rows in float64."""
    f = factor(h.shape[1])
    d = h - h.mean(-1, keepdim=True)
    inv = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    n = d * inv
    lost = f * h.abs().mean(-1, keepdim=True) * inv
    return n, inv, 2 * f * (n.abs() + 1 + lost) + 2 * f * (1 + lost * lost) * n.abs()


def oracle(x, w, b, r, eps):
    """(h, y, y's error before its rounding) on the CPU: h in x's dtype, the others in float64."""
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    n, _, err = stats(h.double(), eps)
    w = torch.ones(x.shape[1], dtype=torch.float64) if w is None else w.double()
    y = n * w
    return h, y if b is None else y + b.double(), err * w.abs() + 2 * U * (y.abs() + (0 if b is None else b.double().abs()))


def oracle_bwd(dy, h, w, dh, eps):
    """(dx, dw, db, dx's error, dw's, db's) in float64."""
    dy, h = dy.double(), h.double()
    f = factor(h.shape[1])
    n, inv, err = stats(h, eps)
    g = dy if w is None else dy * w.double()
    gn = (g * n).mean(-1, keepdim=True)
    dx = inv * (g - g.mean(-1, keepdim=True) - n * gn)
    # g's terms and n's are off by f and err, inv by as much of itself as n is
    size = g.abs() + g.abs().mean(-1, keepdim=True) + n.abs() * gn.abs()
    gn_err = (g.abs() * (err + 2 * f * n.abs())).mean(-1, keepdim=True) + f * (g * n).abs().mean(-1, keepdim=True)
    e = inv * (4 * f * size + n.abs() * gn_err + err * gn.abs() + err * (g.abs() + g.abs().mean(-1, keepdim=True)))
    if dh is not None:
        dx, e = dx + dh.double(), e + U * (dx.abs() + dh.double().abs())
    chain = h.shape[0] * U
    return dx, (dy * n).sum(0), dy.sum(0), e, (dy.abs() * err).sum(0) + 2 * chain * (dy * n).abs().sum(0), chain * dy.abs().sum(0)


def close(got, ref, tol, what):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), f"{what}: NaN in other places"
    over = ((got - ref).abs() - tol).nan_to_num(nan=-1.0)
    assert over.max() <= 0, f"{what}: {over.max().item():.3e} over the tolerance"


def check_fwd(x, w=None, b=None, r=None, eps=1e-5, out8=False, what=""):
    h, y, err = oracle(x, w, b, r, eps)
    dev = [None if t is None else t.to(DEV) for t in (x, w, b, r)]
    got, got_h, scale = _abi.layer_norm_fwd(*dev, eps, torch.float8_e4m3fn if out8 else None)
    torch.cuda.synchronize()
    close(got_h, h.double(), torch.zeros_like(h.double()), what + " h")
    if not out8:
        close(got, y, err + half_step(y, x.dtype), what)
        return
    check_8bit(got.cpu(), scale.cpu(), y, err, what)


def check_8bit(q, scale, y, err, what):
    """8-bit values with block scales against y, known up to err."""
    rows, cols = y.shape
    blocks = -(-cols // 128)

    def tops(t):
        return torch.nn.functional.pad(t, (0, blocks * 128 - cols)).view(rows, blocks, 128).amax(-1)

    top = tops(y.abs())
    s = torch.where(top > 0, top / 448, 1.0)
    close(scale, s, torch.where(top > 0, tops(err) / 448 + 4 * U * s, 0.0), what + " scale")
    s = scale.double().repeat_interleave(128, 1)[:, :cols]
    # half a step of e4m3: 2^-4 of the value, or half the smallest subnormal; the quotient's own rounding
    close(q.float().double() * s, y, err + (2.0 ** -4 + 4 * U) * (y.abs() + err) + 2.0 ** -10 * s, what + " 8 bits")


def check_bwd(dy, h, w=None, dh=None, eps=1e-5, what=""):
    dx, dw, db, e, ew, eb = oracle_bwd(dy, h, w, dh, eps)
    dev = [None if t is None else t.to(DEV) for t in (dy, h, w, dh)]
    got, got_w, got_b = _abi.layer_norm_bwd(*dev, eps=eps)
    torch.cuda.synchronize()
    close(got, dx, e + half_step(dx, h.dtype), what + " dx")
    close(got_w, dw, ew + half_step(dw, got_w.dtype), what + " dw")
    close(got_b, db, eb + half_step(db, got_b.dtype), what + " db")


COLS = [1, 2, 7, 8, 64, 67, 127, 128, 131, 136, 200, 256, 259, 500, 777, 1024, 1031, 2048, 2055, 4096, 4100, 8192, 8197]
LONG = [16384, 16390, 20001]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS + LONG)
def test_forward(gpu, dtype, cols):
    x, w, b = rand((5, cols), dtype, cols, 2.0, 0.3), rand(cols, dtype, 1), rand(cols, dtype, 2)
    r = rand((5, cols), dtype, 3)
    check_fwd(x, w, b, r, what="all")
    check_fwd(x, what="bare")
    check_fwd(x, w, b, r, out8=True, what="to 8 bits")
    check_fwd(x, w.float(), b.float(), out8=True, what="float32 weights")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS + LONG)
def test_backward(gpu, dtype, cols):
    h, dy, w = rand((6, cols), dtype, cols, 2.0, 0.3), rand((6, cols), dtype, 1), rand(cols, dtype, 2, 0.3, 1.0)
    check_bwd(dy, h, w, rand((6, cols), dtype, 4), what="all")
    check_bwd(dy, h, w.float(), what="float32 weights")
    check_bwd(dy, h, what="bare")


@pytest.mark.parametrize("rows,cols", [(1, 256), (33, 256), (300, 777), (1500, 1000), (2100, 96), (5000, 128), (1030, 2048)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(gpu, dtype, rows, cols):
    x, w, b = rand((rows, cols), dtype, rows, 2.0), rand(cols, dtype, 1), rand(cols, dtype, 2)
    check_fwd(x, w, b, what="forward")
    check_fwd(x, w, b, out8=True, what="to 8 bits")
    check_bwd(rand((rows, cols), dtype, 3), x, w, what="backward")


@pytest.mark.parametrize("rows,cols,dtype", [(600, 2100, torch.bfloat16), (700, 4500, torch.float16), (300, 8704, torch.bfloat16),
                                             (600, 5001, torch.float32), (1, 9000, torch.bfloat16)])
def test_many_long_rows(gpu, rows, cols, dtype):
    """Several rows to a workgroup at every length, and one row, whose sums are the gradients themselves."""
    x, w = rand((rows, cols), dtype, rows, 2.0), rand(cols, dtype, 1)
    check_bwd(rand((rows, cols), dtype, 3), x, w, rand((rows, cols), dtype, 4), what="backward")
    check_bwd(rand((rows, cols), dtype, 3), x, w.float(), what="float32 weights")


def test_rows_far_from_zero(gpu):
    """A mean a thousand times the deviation: its rounding is taken off again."""
    for cols in (100, 1000, 5000, 9000):
        x = rand((4, cols), torch.float32, cols, 1.0, 5000.0)
        check_fwd(x, what=f"{cols}")
        check_bwd(rand((4, cols), torch.float32, 1), x, rand(cols, torch.float32, 2), what=f"{cols}")


def test_constant_rows_and_zeros(gpu):
    x = torch.full((3, 130), 7.0)
    x[1] = 0
    check_fwd(x, eps=1e-5, what="constant")
    check_fwd(x, eps=1e-5, out8=True, what="constant, 8 bits")   # zeros: their scale is 1
    check_bwd(rand((3, 130), torch.float32, 1), x, what="constant")


def test_not_numbers(gpu):
    x = rand((3, 300), torch.float16, 0)
    x[0, 5], x[2, 7] = float("nan"), float("inf")
    y, _, _ = _abi.layer_norm_fwd(x.to(DEV))
    y8, _, _ = _abi.layer_norm_fwd(x.to(DEV), out_dtype=torch.float8_e4m3fn)
    dx, _, _ = _abi.layer_norm_bwd(x.to(DEV), x.to(DEV))
    for t in (y, y8.float(), dx):
        assert t[0].isnan().all() and not t[1].isnan().any() and t[2].isnan().all()


def test_strides_and_in_place(gpu):
    cols = 392
    wide = rand((9, 3 * cols + 3), torch.bfloat16, 0).to(DEV)
    x, r, o = wide[:, :cols], wide[:, cols + 3:2 * cols + 3], wide[:, 2 * cols + 3:]
    w, b = rand(cols, torch.bfloat16, 1).to(DEV), rand(cols, torch.bfloat16, 2).to(DEV)
    want, want_h, _ = _abi.layer_norm_fwd(x.contiguous(), w, b, r.contiguous())
    rest = wide[:, cols:cols + 3].clone()
    out = torch.empty((9, cols), dtype=torch.bfloat16, device=DEV)
    d = _abi.make_layer_norm_desc(x, w, b, o, r, r, stream=torch.cuda.current_stream().cuda_stream)
    _abi.check(_abi.load().tvk_layer_norm_fwd(_abi.C.byref(d)))   # h over the residual
    assert torch.equal(o, want) and torch.equal(r, want_h) and torch.equal(wide[:, cols:cols + 3], rest)
    d = _abi.make_layer_norm_desc(r, w, b, r, stream=torch.cuda.current_stream().cuda_stream)
    _abi.check(_abi.load().tvk_layer_norm_fwd(_abi.C.byref(d)))   # in place
    assert torch.equal(r, _abi.layer_norm_fwd(want_h, w, b)[0])
    # scales in columns of their own, 8-bit rows at odd places
    q = torch.zeros((9, cols + 5), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    s = torch.zeros((4, 9), device=DEV)
    d = _abi.make_layer_norm_desc(out.copy_(x), w, b, q[:, 3:cols + 3], scale=s.t(), stream=torch.cuda.current_stream().cuda_stream)
    _abi.check(_abi.load().tvk_layer_norm_fwd(_abi.C.byref(d)))
    want8, _, want_s = _abi.layer_norm_fwd(out, w, b, out_dtype=torch.float8_e4m3fn)
    u8 = q.view(torch.uint8)
    assert torch.equal(u8[:, 3:cols + 3], want8.view(torch.uint8)) and torch.equal(s.t(), want_s)
    assert not u8[:, :3].any() and not u8[:, cols + 3:].any()


def test_backward_in_place_and_what_is_wanted(gpu):
    for cols, rows in ((500, 40), (20000, 3)):
        dy, h = rand((rows, cols), torch.float32, 1).to(DEV), rand((rows, cols), torch.float32, 2).to(DEV)
        w = rand(cols, torch.float32, 3).to(DEV)
        dx, dw, db = _abi.layer_norm_bwd(dy, h, w)
        for want_w, want_b in ((True, False), (False, True), (False, False)):
            for over in (dy, h):
                src = [dy.clone(), h.clone()]
                to = src[0] if over is dy else src[1]
                gw, gb = torch.full_like(w, 9.0), torch.full_like(w, 9.0)
                d = _abi.make_layer_norm_bwd_desc(*src, w, to, gw if want_w else None, gb if want_b else None,
                                                  stream=torch.cuda.current_stream().cuda_stream)
                _abi.check(_abi.load().tvk_layer_norm_bwd(_abi.C.byref(d)))
                assert torch.equal(to, dx)
                assert torch.equal(gw, dw if want_w else torch.full_like(w, 9.0))
                assert torch.equal(gb, db if want_b else torch.full_like(w, 9.0))


def test_no_rows(gpu):
    w = torch.ones(64, device=DEV)
    empty = torch.empty((0, 64), device=DEV)
    dx, dw, db = _abi.layer_norm_bwd(empty, empty, w)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()
    assert _abi.layer_norm_fwd(empty, w)[0].shape == (0, 64)


def test_captured(gpu):
    """Replays of a captured forward and backward, with eager calls between them, give the eager call's bits."""
    h, dy, w = (rand(s, torch.bfloat16, i).to(DEV) for i, s in enumerate(((700, 1000), (700, 1000), (1000,))))
    _abi.layer_norm_bwd(dy, h, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _, _ = _abi.layer_norm_fwd(h, w, w)
        out = _abi.layer_norm_bwd(dy, h, w)
    for i in range(3):
        h.copy_(rand((700, 1000), torch.bfloat16, 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, *out)]
        want = [_abi.layer_norm_fwd(h, w, w)[0], *_abi.layer_norm_bwd(dy, h, w)]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_autograd(gpu):
    """decoder.layer_norm on the vulkan device: the gradients that its formula gives, for every input that wants one."""
    x, r, g1, g2 = (rand((2, 6, 96), torch.float32, i) for i in range(4))
    w, b = rand(96, torch.float32, 5), rand(96, torch.float32, 6)
    leaves = [t.to("vulkan").requires_grad_() for t in (x, w, b, r)]
    y, h = decoder.layer_norm(leaves[0], leaves[1], leaves[2], leaves[3])
    torch.autograd.backward([y, h], [g1.to("vulkan"), g2.to("vulkan")])
    hh = (x + r).view(-1, 96)
    dx, dw, db, e, ew, eb = oracle_bwd(g1.view(-1, 96), hh, w, g2.view(-1, 96), 1e-5)
    for leaf, ref, err in ((leaves[0], dx, e), (leaves[3], dx, e), (leaves[1], dw, ew), (leaves[2], db, eb)):
        close(leaf.grad.cpu().view(ref.shape), ref, err + half_step(ref, torch.float32), "autograd")
    only = b.to("vulkan").requires_grad_()
    decoder.layer_norm(x.to("vulkan"), None, only).sum().backward()
    close(only.grad.cpu(), torch.full((96,), 12.0, dtype=torch.float64), 12 * U * 12, "bias alone")
    q, s, h = decoder.layer_norm_fp8(leaves[0], leaves[1])
    assert s.shape == (2, 6, 1) and h is leaves[0]
    with pytest.raises(_abi.TvkUnsupported):
        s.sum().backward()
