"""tvk_quantize_f8 and tvk_gemm_f8 against their formulas.

The 8-bit values are compared bit for bit: a scale is one float32 division, its
reciprocal another, a value one product rounded to e4m3, all of which the CPU
does alike. Products are compared in float64: a block's sum of 128 products runs
in the matrix unit, in at most 128 additions, the blocks' sums in one
multiply-add each, and the waves' in 8: with u = 2^-24 the result is off by at
most 2 (128 + blocks + 16) u of the sum of its terms' magnitudes. For a 16-bit
output the matrix unit cuts each of eight neighbouring products off at 2^-13 of
the power of two at or below their largest: seven of them lose less than 2^-13 of the
largest each, which is at most the largest |a| times the largest |b| of those
eight. The result's rounding adds half a step of its type (eps / 2 of the value,
or half the smallest subnormal)."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from torchvulkan_amd import _abi, decoder

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
F8 = torch.float8_e4m3fn
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def rand(shape, seed, std=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std


def quantized(x, tall=1):
    """(values, scale) of float32 x, on the CPU."""
    rows, cols = x.shape
    x = x.float()
    p = torch.nn.functional.pad(x, (0, -cols % 128, 0, -rows % tall))
    t = p.view(-1, tall, p.shape[1] // 128, 128)
    top = t.abs().nan_to_num(nan=0.0, posinf=math.inf).amax((1, 3))
    scale = torch.where(top > 0, top / 448, 1.0)
    r = 1 / scale
    plain = (r < 1e30) & (r > 1e-30)
    q = torch.where(plain[:, None, :, None], t * r[:, None, :, None], t / scale[:, None, :, None])
    return q.reshape(p.shape)[:rows, :cols].to(F8), scale


def bits(t):
    return t.cpu().view(torch.uint8)


def spread(scale, tall, rows, cols):
    return scale.double().repeat_interleave(tall, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def check(a, sa, b, sb, bias=None, out_dtype=torch.float32, what="", dev=None):
    """dev: a, sa, b, sb as the call gets them (layouts of their own), else contiguous."""
    m, k = a.shape
    x = a.double() * spread(sa, 1, m, k)
    w = b.double() * spread(sb, 128, b.shape[0], k)
    x, w = x.to(DEV), w.to(DEV)
    ref, size = torch.matmul(x, w.t().contiguous()), torch.matmul(x.abs(), w.t().contiguous().abs())
    if bias is not None:
        ref, size = ref + bias.double().to(DEV), size + bias.double().abs().to(DEV)
    got = _abi.gemm_f8(*(dev or [t.to(DEV) for t in (a, sa, b, sb)]), None if bias is None else bias.to(DEV), out_dtype)
    torch.cuda.synchronize()
    assert got.dtype == out_dtype
    tol = 2 * (128 + -(-k // 128) + 16) * U * size
    if out_dtype != torch.float32:
        eights = [torch.nn.functional.pad(t.abs(), (0, -k % 8)).view(t.shape[0], -1, 8).amax(-1) for t in (x, w)]
        tol += 7 * 2.0 ** -13 * torch.matmul(eights[0], eights[1].t().contiguous())
    tol += torch.finfo(out_dtype).eps / 2 * ref.abs() + TINY[out_dtype]
    over = ((got.double() - ref).abs() - tol).max().item()
    assert over <= 0, f"{what}: {over:.3e} over the tolerance"
    return got


def operands(m, n, k, seed):
    return *quantized(rand((m, k), seed) * torch.exp(rand((k,), seed + 1))), *quantized(rand((n, k), seed + 2, 0.1), 128)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 127), (2, 128), (5, 129), (130, 300), (257, 1000), (40, 4099)])
def test_quantize(gpu, dtype, rows, cols):
    x = (rand((rows, cols), rows) * 5).to(dtype)
    x[0, :] = 0
    for tall in (1, 128):
        q, s = _abi.quantize_f8(x.to(DEV), tall)
        want, scale = quantized(x, tall)
        assert torch.equal(s.cpu(), scale) and torch.equal(bits(q), bits(want))


def test_quantize_ends_of_the_range(gpu):
    x = rand((6, 256), 0)
    x[0] *= 1e38
    x[1] *= 1e-38
    x[2] *= 1e-44
    x[3, 7], x[4, 9], x[4, 200] = math.nan, math.inf, -math.nan
    q, s = _abi.quantize_f8(x.to(DEV))
    want, scale = quantized(x)
    assert torch.equal(s.cpu(), scale)
    a, b = q.cpu().float(), want.float()
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def test_quantize_strides(gpu):
    x = rand((9, 500), 3).half()
    want, scale = quantized(x[:, 3:303])
    out, s = torch.zeros((9, 400), dtype=torch.uint8, device=DEV).view(F8), torch.zeros((3, 9), device=DEV)
    d = _abi.make_quantize_f8_desc(x.to(DEV)[:, 3:303], out[:, 5:305], s.t(), 1, torch.cuda.current_stream().cuda_stream)
    _abi.check(_abi.load().tvk_quantize_f8(C.byref(d)))
    b = bits(out)
    assert torch.equal(s.t().cpu(), scale) and torch.equal(b[:, 5:305], bits(want)) and not b[:, :5].any() and not b[:, 305:].any()


@pytest.mark.parametrize("m", [1, 3, 16, 17, 32, 33, 64, 65, 128, 130, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (15, 100), (16, 128), (130, 129), (200, 16), (500, 1000), (129, 4112), (256, 2048)])
def test_sizes(gpu, m, n, k):
    check(*operands(m, n, k, m + n + k), what=f"{m} {n} {k}")


@pytest.mark.parametrize("m,n,k", [(4100, 4097, 256), (4096, 4352, 400), (1000, 9000, 1040), (2048, 2048, 1024)])
def test_large(gpu, m, n, k):
    """Tiles of 256 x 256, whole and cut."""
    check(*operands(m, n, k, 1), out_dtype=torch.bfloat16)


@pytest.mark.parametrize("m,n,k", [(2048, 4096, 144), (2000, 4000, 640), (1400, 4200, 400)])
def test_middling(gpu, m, n, k):
    """Tiles of 128 x 256, whole and cut, of one step and of several."""
    for dtype in (torch.bfloat16, torch.float16):
        check(*operands(m, n, k, 2), bias=rand((n,), 3), out_dtype=dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [2, 50, 200])
def test_types_and_bias(gpu, dtype, m):
    a, sa, b, sb = operands(m, 333, 700, m)
    check(a, sa, b, sb, rand((333,), 5), dtype, "float32 bias")
    check(a, sa, b, sb, rand((333,), 6).to(dtype), dtype, "bias")


@pytest.mark.parametrize("m", [1, 4, 5, 16, 32, 64])
@pytest.mark.parametrize("n,k", [(40, 5), (40, 15), (40, 17), (40, 31), (40, 143), (4097, 300), (6145, 300), (8200, 400), (12300, 700)])
def test_few_rows(gpu, m, n, k):
    """Ends of rows at every part of 16 bytes, and columns enough for several blocks of W a workgroup; wider rows give the
    bits of their 8-bit form."""
    for out_dtype in (torch.float32, torch.bfloat16):
        check(*operands(m, n, k, m + k), out_dtype=out_dtype, what=f"{m} {n} {k}")
    _, _, b, sb = operands(1, n, k, k)
    for dtype in DTYPES:
        a = (rand((m, k), k) * 3).to(dtype).to(DEV)
        q, sa = _abi.quantize_f8(a)
        want = _abi.gemm_f8(q, sa, b.to(DEV), sb.to(DEV), out_dtype=dtype)
        assert torch.equal(_abi.gemm_f8(a, None, b.to(DEV), sb.to(DEV)), want)


@pytest.mark.parametrize("m,n,k", [(17, 12290, 4096), (17, 2100, 15440), (32, 4100, 12288), (33, 2100, 4096), (33, 300, 8192), (64, 4096, 2064), (64, 4096, 4112)])
def test_few_rows_of_large_weights(gpu, m, n, k):
    a, sa, b, sb = operands(m, n, k, m)
    for out_dtype in (torch.float32, torch.float16):
        check(a, sa, b, sb, out_dtype=out_dtype, what="aligned")
    wide = torch.zeros((n, k + 16), dtype=torch.uint8, device=DEV).view(F8)   # rows that 16-byte loads do not meet
    wide[:, 3:k + 3] = b.to(DEV)
    check(a, sa, b, sb, out_dtype=torch.float16, what="unaligned", dev=[a.to(DEV), sa.to(DEV), wide[:, 3:k + 3], sb.to(DEV)])
    x = (a.float() * 3).bfloat16().to(DEV)
    q, sx = _abi.quantize_f8(x)
    assert torch.equal(_abi.gemm_f8(x, None, b.to(DEV), sb.to(DEV)), _abi.gemm_f8(q, sx, b.to(DEV), sb.to(DEV)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 100, 300), (7, 33, 4100), (16, 512, 128), (17, 130, 700), (64, 64, 1), (70, 200, 333), (300, 300, 512)])
def test_rows_in_more_bits(gpu, dtype, m, n, k):
    """The call's own 8 bits are tvk_quantize_f8's: the same product, bit for bit."""
    x = (rand((m, k), m) * 3).to(dtype)
    b, sb = quantized(rand((n, k), 9), 128)
    q, sq = quantized(x)
    want = check(q, sq, b, sb, out_dtype=dtype)
    got = _abi.gemm_f8(x.to(DEV), None, b.to(DEV), sb.to(DEV))
    assert torch.equal(got, want)


@pytest.mark.parametrize("m", [5, 40, 200])
def test_every_8_bit_value(gpu, m):
    """Each of the 254 numbers times one, in both kinds of sums."""
    codes = torch.tensor([c for c in range(256) if c & 127 != 127], dtype=torch.uint8)
    b = torch.zeros((254, 5), dtype=torch.uint8)
    b[:, 3] = codes
    a = torch.ones((m, 5)).to(F8)
    one = torch.ones((m, 1)), torch.ones((2, 1))
    for dtype in (torch.float32, torch.float16):
        got = _abi.gemm_f8(a.to(DEV), one[0].to(DEV), b.view(F8).to(DEV), one[1].to(DEV), out_dtype=dtype)
        assert torch.equal(got.cpu(), codes.view(F8).to(dtype).expand(m, 254))


@pytest.mark.parametrize("m", [5, 40, 200])
def test_layouts(gpu, m):
    """Rows at odd places of wider ones whose other bytes are NaN, scales in columns, one scale for all."""
    a, sa, b, sb = operands(m, 300, 400, m)
    wide_a = torch.full((m + 1, 480), 0x7f, dtype=torch.uint8, device=DEV).view(F8)
    wide_b = torch.full((301, 500), 0xff, dtype=torch.uint8, device=DEV).view(F8)
    va, vb = wide_a[:m, 16:416], wide_b[:300, 7:407]
    va.view(torch.uint8).copy_(a.view(torch.uint8))
    vb.view(torch.uint8).copy_(b.view(torch.uint8))
    ca, cb = sa.t().contiguous().to(DEV).t(), sb.t().contiguous().to(DEV).t()
    want = check(a, sa, b, sb)
    assert torch.equal(check(a, sa, b, sb, dev=[va, ca, vb, cb]), want)
    out = torch.zeros((m, 310), device=DEV)
    d = _abi.make_gemm_f8_desc(va, ca, vb, cb, out[:, 3:303], stream=torch.cuda.current_stream().cuda_stream)
    _abi.check(_abi.load().tvk_gemm_f8(C.byref(d)))
    assert torch.equal(out[:, 3:303], want) and not out[:, :3].any() and not out[:, 303:].any()
    one = torch.full((1, 1), 0.5)
    check(a, one.expand(m, 4), b, one.expand(3, 4), dev=[a.to(DEV), one.to(DEV).expand(m, 4), b.to(DEV), one.to(DEV).expand(3, 4)])
    row = a[:1].to(DEV).expand(m, 400)   # one row for all
    check(a[:1].expand(m, 400), sa, b, sb, dev=[row, sa.to(DEV), b.to(DEV), sb.to(DEV)])


@pytest.mark.parametrize("m", [4, 40, 130])
def test_not_numbers_stay_where_they_are(gpu, m):
    """NaN, an infinite scale and odd ends of k touch the outputs that they belong to and no others."""
    n, k = 150, 200
    a, sa, b, sb = operands(m, n, k, m)
    want = _abi.gemm_f8(*(t.to(DEV) for t in (a, sa, b, sb)), out_dtype=torch.float32)
    a2, b2, sa2 = a.view(torch.uint8).clone(), b.view(torch.uint8).clone(), sa.clone()
    a2[2, 199], b2[77, 0], sa2[3, 1] = 0x7f, 0xff, math.inf
    got = _abi.gemm_f8(a2.view(F8).to(DEV), sa2.to(DEV), b2.view(F8).to(DEV), sb.to(DEV), out_dtype=torch.float32)
    bad = torch.zeros((m, n), dtype=torch.bool, device=DEV)
    bad[2], bad[3], bad[:, 77] = True, True, True
    assert torch.equal(got[~bad], want[~bad])
    assert got[2].isnan().all() and got[:, 77].isnan().all() and not got[3].isfinite().any()


def test_nothing(gpu):
    for m, n, k in ((0, 5, 9), (5, 0, 9), (3, 20, 0), (70, 20, 0)):
        a, b = torch.zeros((m, k), device=DEV).to(F8), torch.zeros((n, k), device=DEV).to(F8)
        blocks = -(-k // 128)
        bias = torch.arange(n, device=DEV, dtype=torch.float32)
        out = _abi.gemm_f8(a, torch.zeros((m, blocks), device=DEV), b, torch.zeros((-(-n // 128), blocks), device=DEV), bias, torch.float32)
        assert torch.equal(out, bias.expand(m, n))


def test_captured(gpu):
    """Replays of captured products that lay rows out in scratch, with eager calls between them, give the eager call's bits."""
    b, sb = (t.to(DEV) for t in quantized(rand((300, 333), 1), 128))
    xs = [rand((m, 333), m).bfloat16().to(DEV) for m in (3, 40, 100)]
    for x in xs:
        _abi.gemm_f8(x, None, b, sb)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [_abi.gemm_f8(x, None, b, sb) for x in xs]
    for i in range(3):
        for x in xs:
            x.copy_(rand(tuple(x.shape), 50 + i).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(g, _abi.gemm_f8(x, None, b, sb)) for g, x in zip(got, xs))


@pytest.mark.parametrize("device", ["cuda", "vulkan"])
def test_linear(gpu, device):
    """layer norm to 8 bits, an 8-bit weight made on the device, and their product: the composition in float64, with the
    8-bit values' own steps in its tolerance (2^-4 of a value and of the block's scale 2^-10, for either factor)."""
    x, w = rand((2, 5, 300), 1), rand((70, 300), 2, 0.1)
    q, s = decoder.quantize_fp8(w.to(device), 128)
    y8, ys, _ = decoder.layer_norm_fp8(x.to(device))
    got = decoder.linear_fp8(y8, q, s, x_scale=ys, out_dtype=torch.float32)
    assert got.shape == (2, 5, 70)
    y = torch.nn.functional.layer_norm(x.double(), (300,)).view(10, 300)
    ref, top = y @ w.double().t(), 448.0
    dy = y.abs() * 2.0 ** -4 + 2.0 ** -10 * y.abs().max() / top + 1e-6
    dw = w.double().abs() * 2.0 ** -4 + 2.0 ** -10 * w.abs().max() / top
    tol = (y.abs() + dy) @ dw.t() + dy @ w.double().abs().t() + 1e-5
    assert ((got.cpu().double().view(10, 70) - ref).abs() <= tol).all()
    again = decoder.linear_fp8(x.to(device), q, s)
    assert again.dtype == torch.float32 and again.shape == (2, 5, 70)
    leaf = x.to(device).requires_grad_()
    with pytest.raises((_abi.TvkUnsupported, RuntimeError)):
        decoder.linear_fp8(leaf, q, s).sum().backward()
