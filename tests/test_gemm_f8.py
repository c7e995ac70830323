"""CPU checks of the 8-bit block products: what their entry points refuse."""
import ctypes as C

import pytest
import torch

from torchvulkan_amd import _abi, decoder

lib = _abi.load()
I2 = _abi.I64x2
F8 = torch.float8_e4m3fn


def status(fn, desc):
    st = getattr(lib, fn)(C.byref(desc))
    assert st == _abi.TVK_OK or fn.encode() in lib.tvk_last_error()
    return _abi.STATUS_NAMES[st]


def gemm(**kw):
    d = _abi.GemmF8Desc()
    d.a_dtype, d.out_dtype, d.bias_dtype = _abi.TVK_F8E4M3FN, _abi.TVK_BF16, _abi.TVK_BF16
    d.M, d.N, d.K = 4, 300, 200
    d.a = d.b = d.a_scale = d.b_scale = d.out = 16   # never dereferenced by validation
    d.a_stride = d.b_stride = 200
    d.a_scale_stride = d.b_scale_stride = I2(2, 1)
    d.out_stride = 300
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,want", [
    ({"a_dtype": _abi.TVK_F8E5M2}, "UNSUPPORTED"), ({"a_dtype": _abi.TVK_F64}, "UNSUPPORTED"), ({"out_dtype": _abi.TVK_F8E4M3FN}, "UNSUPPORTED"),
    ({"bias_dtype": _abi.TVK_F16}, "UNSUPPORTED"), ({"M": -1}, "INVALID"), ({"N": -1}, "INVALID"), ({"K": -1}, "INVALID"),
    ({"M": 1 << 31}, "UNSUPPORTED"), ({"N": 1 << 31}, "UNSUPPORTED"), ({"K": (1 << 31) - 1}, "UNSUPPORTED"),
    ({"M": 65, "K": (1 << 22) + 1}, "UNSUPPORTED"), ({"M": 1 << 20, "N": 1 << 20, "out_stride": 1 << 20}, "UNSUPPORTED"),
    ({"a": None}, "INVALID"), ({"b": None}, "INVALID"), ({"out": None}, "INVALID"), ({"a_scale": None}, "INVALID"),
    ({"b_scale": None}, "INVALID"), ({"a_stride": -1}, "INVALID"), ({"b_stride": -1}, "INVALID"), ({"out_stride": 299}, "INVALID"),
    ({"a_scale_stride": I2(-1, 1)}, "INVALID"), ({"b_scale_stride": I2(1, -1)}, "INVALID"), ({"M": 0}, "OK"), ({"N": 0, "b": None}, "OK"),
])
def test_refusals(kw, want):
    assert status("tvk_gemm_f8", gemm(**kw)) == want


def quantize(**kw):
    d = _abi.QuantizeF8Desc()
    d.dtype, d.block_rows = _abi.TVK_F16, 1
    d.rows, d.cols = 300, 200
    d.x = d.out = d.scale = 16
    d.x_stride = d.out_stride = 200
    d.scale_stride = I2(2, 1)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,want", [
    ({"dtype": _abi.TVK_F64}, "UNSUPPORTED"), ({"block_rows": 64}, "UNSUPPORTED"), ({"block_rows": 0}, "UNSUPPORTED"), ({"rows": -1}, "INVALID"),
    ({"cols": -1}, "INVALID"), ({"rows": 1 << 31}, "UNSUPPORTED"), ({"cols": 1 << 31}, "UNSUPPORTED"), ({"x": None}, "INVALID"),
    ({"out": None}, "INVALID"), ({"scale": None}, "INVALID"), ({"x_stride": -1}, "INVALID"), ({"out_stride": 199}, "INVALID"),
    ({"scale_stride": I2(1, 1)}, "INVALID"), ({"scale_stride": I2(0, 1)}, "INVALID"), ({"scale_stride": I2(1, 299)}, "INVALID"),
    ({"rows": 0}, "OK"), ({"cols": 0, "x": None}, "OK"),
])
def test_quantize_refusals(kw, want):
    assert status("tvk_quantize_f8", quantize(**kw)) == want


def test_null_descriptors():
    for fn in ("tvk_gemm_f8", "tvk_quantize_f8"):
        assert getattr(lib, fn)(None) == _abi.TVK_ERR_INVALID
        assert fn.encode() in lib.tvk_last_error()


def test_binding_refuses_other_layouts():
    a, b, h = torch.zeros((3, 200)).to(F8), torch.zeros((300, 200)).to(F8), torch.zeros((3, 200), dtype=torch.float16)
    sa, sb, out = torch.zeros((3, 2)), torch.zeros((3, 2)), torch.zeros((3, 300), dtype=torch.bfloat16)
    make, quant = _abi.make_gemm_f8_desc, _abi.make_quantize_f8_desc
    make(a, sa, b, sb, out)
    make(a, torch.zeros((2, 3)).t(), b, sb[:1].expand(3, 2), out, bias=torch.zeros(300))
    make(h, None, b, sb, out, bias=out[0])
    quant(h, a, sa)
    quant(b.float(), b, sb, 128)
    for bad in (lambda: make(a, None, b, sb, out), lambda: make(h, sa, b, sb, out), lambda: make(a, sa[:2], b, sb, out),
                lambda: make(a, sa, b, sb[:2], out), lambda: make(a, sa, b, sb.double(), out), lambda: make(a, sa, b[:, :199], sb, out),
                lambda: make(a, sa, b.float(), sb, out), lambda: make(a, sa, b, sb, out[:, :299]), lambda: make(a, sa, b, sb, out, out[0][:9]),
                lambda: make(a[0], sa, b, sb, out), lambda: make(a, sa, b, sb, out, torch.zeros(300).half()),
                lambda: make(a, sa, b, sb, out.double()), lambda: quant(h, a, sb, 128), lambda: quant(h, h, sa), lambda: quant(h, a, sa, 64),
                lambda: decoder.linear_fp8(a, b, sb, x_scale=sa[:2]), lambda: decoder.linear_fp8(h, b, sb),
                lambda: decoder.quantize_fp8(h), lambda: decoder.quantize_fp8(h[None], 128)):
        with pytest.raises(_abi.TvkError):
            bad()
