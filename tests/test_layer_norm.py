"""CPU checks of layer norm: what its entry points refuse, and its backward
formula (the GPU tests' oracle) against differences of the forward."""
import ctypes as C

import pytest
import torch

from torchvulkan_amd import _abi, decoder

lib = _abi.load()
I2 = _abi.I64x2


def status(fn, desc):
    st = getattr(lib, fn)(C.byref(desc))
    assert st == _abi.TVK_OK or fn.encode() in lib.tvk_last_error()
    return _abi.STATUS_NAMES[st]


def norm(**kw):
    d = _abi.LayerNormDesc()
    d.dtype = d.out_dtype = d.weight_dtype = _abi.TVK_F16
    d.rows, d.cols = 4, 300
    d.x = d.out = d.weight = d.bias = 16   # never dereferenced by validation
    d.x_stride = d.out_stride = 300
    d.eps = 1e-5
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def in8(**kw):
    return {"out_dtype": _abi.TVK_F8E4M3FN, "scale": 16, "scale_stride": I2(3, 1), **kw}


@pytest.mark.parametrize("kw,want", [
    ({"dtype": _abi.TVK_F64}, "UNSUPPORTED"), ({"out_dtype": _abi.TVK_F32}, "UNSUPPORTED"),
    ({"out_dtype": _abi.TVK_F8E5M2}, "UNSUPPORTED"), ({"weight_dtype": _abi.TVK_BF16}, "UNSUPPORTED"),
    ({"rows": -1}, "INVALID"), ({"cols": -1}, "INVALID"), ({"eps": -1.0}, "INVALID"), ({"eps": float("nan")}, "INVALID"),
    ({"x": None}, "INVALID"), ({"out": None}, "INVALID"), ({"x_stride": -300}, "INVALID"), ({"out_stride": 299}, "INVALID"),
    ({"residual": 16, "residual_stride": -1}, "INVALID"), ({"residual_out": 16, "residual_out_stride": 0}, "INVALID"),
    (in8(scale=None), "INVALID"), (in8(scale_stride=I2(2, 1)), "INVALID"), (in8(scale_stride=I2(3, 0)), "INVALID"),
    (in8(scale_stride=I2(-3, 1)), "INVALID"), (in8(scale_stride=I2(1, 3)), "INVALID"),
    ({"rows": 1 << 31}, "UNSUPPORTED"), ({"cols": 1 << 31}, "UNSUPPORTED"), ({"rows": 0, "x": None}, "OK"),
    ({"cols": 0}, "OK"), (in8(rows=0), "OK"),
])
def test_refusals(kw, want):
    assert status("tvk_layer_norm_fwd", norm(**kw)) == want


def bwd(**kw):
    d = _abi.LayerNormBwdDesc()
    d.dtype = d.weight_dtype = _abi.TVK_BF16
    d.rows, d.cols = 4, 64
    d.dy = d.h = d.dx = d.weight = d.dweight = d.dbias = 16
    d.dy_stride = d.h_stride = d.dx_stride = 64
    d.eps = 1e-5
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,want", [
    ({"dtype": _abi.TVK_I8}, "UNSUPPORTED"), ({"weight_dtype": _abi.TVK_F16}, "UNSUPPORTED"), ({"rows": -2}, "INVALID"),
    ({"dy": None}, "INVALID"), ({"h": None}, "INVALID"), ({"dx": None}, "INVALID"), ({"dx_stride": 1}, "INVALID"),
    ({"dh": 16, "dh_stride": -64}, "INVALID"), ({"eps": -1e-9}, "INVALID"), ({"cols": 0}, "OK"),
    ({"rows": 0, "dweight": None, "dbias": None}, "OK"),
])
def test_bwd_refusals(kw, want):
    assert status("tvk_layer_norm_bwd", bwd(**kw)) == want


def test_null_descriptors():
    for fn in ("tvk_layer_norm_fwd", "tvk_layer_norm_bwd"):
        assert getattr(lib, fn)(None) == _abi.TVK_ERR_INVALID
        assert fn.encode() in lib.tvk_last_error()


def test_binding_refuses_other_layouts():
    h = torch.float16
    x, w = torch.zeros((4, 200), dtype=h), torch.zeros(200, dtype=h)
    out8, scale = torch.zeros((4, 200), dtype=torch.float8_e4m3fn), torch.zeros((4, 2))
    make, back = _abi.make_layer_norm_desc, _abi.make_layer_norm_bwd_desc
    make(x, w, w, x)
    make(x, w, None, out8, scale=scale)
    make(x, None, w.float(), out8, scale=torch.zeros((2, 4)).t())
    back(x, x, w, x, w, w)
    for bad in (lambda: make(x, w[:7], None, x), lambda: make(x, w, w.float(), x), lambda: make(x, w, w, out8),
                lambda: make(x, w, w, x, scale=scale), lambda: make(x, w, w, out8, scale=scale[:3]),
                lambda: make(x, w, w, out8, scale=scale.double()), lambda: make(x, w.double(), w, x),
                lambda: make(x, w, w, x, residual=x[:2]), lambda: make(x.t(), None, None, x.t()), lambda: make(x[0], w, w, x),
                lambda: back(x, x, w, x, w.float()), lambda: back(x, x, w, x, w, w.float()), lambda: back(x.float(), x, w, x, w)):
        with pytest.raises(_abi.TvkError):
            bad()
    with pytest.raises(_abi.TvkError):
        decoder.layer_norm(x, w, w)   # on the host
    with pytest.raises(_abi.TvkError):
        decoder.layer_norm(x, w, w, residual=x.float())


def test_backward_formula():
    """The formula of the gradients, and with it the GPU tests' oracle, against central differences: their error is of
    order step^2, 1e-10 here, and cancellation's 1e-16 / step."""
    from tests.test_layer_norm_gpu import oracle_bwd

    g = torch.Generator().manual_seed(0)
    x, dy, dh = (torch.randn((3, 11), generator=g, dtype=torch.float64) for _ in range(3))
    w, b = torch.randn(11, generator=g, dtype=torch.float64), torch.randn(11, generator=g, dtype=torch.float64)
    eps, step = 1e-3, 1e-5

    def value(x, w, b):
        d = x - x.mean(-1, keepdim=True)
        return ((d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps) * w + b) * dy).sum() + (x * dh).sum()

    got = oracle_bwd(dy, x, w, dh, eps)
    for t, grad in ((x, got[0]), (w, got[1]), (b, got[2])):
        for i in range(t.numel()):
            d = torch.zeros(t.numel(), dtype=torch.float64)
            d[i] = step
            up, down = (value(*[v + s * d.view(v.shape) if v is t else v for v in (x, w, b)]) for s in (1, -1))
            assert abs((up - down) / (2 * step) - grad.flatten()[i]) < 1e-8
