"""CPU checks of the distillation loss: what its entry points refuse, and its
gradient's formula (the GPU tests' oracle) against differences of the loss."""
import ctypes as C

import pytest
import torch

from torchvulkan_amd import _abi, decoder

lib = _abi.load()


def status(fn, desc):
    st = getattr(lib, fn)(C.byref(desc))
    assert st == _abi.TVK_OK or fn.encode() in lib.tvk_last_error()
    return _abi.STATUS_NAMES[st]


def filled(cls, kw):
    d = cls()
    d.dtype = _abi.TVK_BF16
    d.index_dtype = _abi.TVK_I64
    d.rows, d.cols, d.top = 4, 1000, 8
    d.logits = d.index = d.lse = d.target = 16   # never dereferenced by validation
    d.logits_stride, d.index_stride, d.target_stride = 1000, 8, 8
    if cls is _abi.DistillDesc:
        d.teacher_dtype, d.teacher, d.teacher_stride, d.loss = _abi.TVK_F32, 16, 8, 16
    else:
        d.dloss, d.dloss_stride, d.dlogits, d.dlogits_stride = 16, 1, 16, 1000
    d.temperature = 1.0
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BOTH = [
    ({"dtype": _abi.TVK_F64}, "UNSUPPORTED"), ({"index_dtype": _abi.TVK_I16}, "UNSUPPORTED"), ({"rows": -1}, "INVALID"),
    ({"cols": -1}, "INVALID"), ({"top": -1}, "INVALID"), ({"top": 2049}, "UNSUPPORTED"), ({"rows": 1 << 31}, "UNSUPPORTED"),
    ({"cols": 1 << 31}, "UNSUPPORTED"), ({"temperature": 0.0}, "INVALID"), ({"temperature": -1.0}, "INVALID"),
    ({"temperature": float("nan")}, "INVALID"), ({"temperature": float("inf")}, "INVALID"), ({"temperature": 1e-40}, "INVALID"),
    ({"temperature": 1e30}, "INVALID"), ({"logits": None}, "INVALID"), ({"index": None}, "INVALID"),
    ({"logits_stride": -1}, "INVALID"), ({"index_stride": -8}, "INVALID"), ({"rows": 0}, "OK"),
]


@pytest.mark.parametrize("kw,want", BOTH + [
    ({"teacher_dtype": _abi.TVK_F16}, "UNSUPPORTED"), ({"teacher": None}, "INVALID"), ({"loss": None}, "INVALID"),
    ({"teacher_stride": -1}, "INVALID"), ({"target_stride": 7}, "INVALID"),
])
def test_refusals(kw, want):
    assert status("tvk_distill_fwd", filled(_abi.DistillDesc, kw)) == want


@pytest.mark.parametrize("kw,want", BOTH + [
    ({"lse": None}, "INVALID"), ({"target": None}, "INVALID"), ({"dloss": None}, "INVALID"), ({"dlogits": None}, "INVALID"),
    ({"dloss_stride": -1}, "INVALID"), ({"target_stride": -1}, "INVALID"), ({"dlogits_stride": 999}, "INVALID"), ({"cols": 0}, "OK"),
])
def test_bwd_refusals(kw, want):
    assert status("tvk_distill_bwd", filled(_abi.DistillBwdDesc, kw)) == want


def test_null_descriptors():
    for fn in ("tvk_distill_fwd", "tvk_distill_bwd"):
        assert getattr(lib, fn)(None) == _abi.TVK_ERR_INVALID
        assert fn.encode() in lib.tvk_last_error()


def test_binding_refuses_other_layouts():
    x, i, t = torch.zeros((3, 50), dtype=torch.float16), torch.zeros((3, 4), dtype=torch.int32), torch.zeros((3, 4))
    v, q = torch.zeros(3), torch.zeros((3, 4))
    make, back = _abi.make_distill_desc, _abi.make_distill_bwd_desc
    make(x, i, t, v, v, q)
    back(x, i, v, q, v[:1].expand(3), x)
    for bad in (lambda: make(x[0], i, t, v), lambda: make(x, i[:2], t, v), lambda: make(x, i.short(), t, v),
                lambda: make(x, i, t.double(), v), lambda: make(x, i, t[:, :3], v), lambda: make(x, i, t, v.double()),
                lambda: make(x, i, t, v, v[:2]), lambda: make(x, i, t, v, v, q.t()), lambda: make(x.t(), i, t, v),
                lambda: back(x, i, v, q, v[:2], x), lambda: back(x, i, v, q, v, x.float()), lambda: back(x, i, v, q.double(), v, x)):
        with pytest.raises(_abi.TvkError):
            bad()
    for bad in (lambda: decoder.distill_loss(x, i, t), lambda: decoder.distill_loss(x, i, t[:, :2]),
                lambda: decoder.distill_loss(x[0], i, t)):   # on the host; lists that do not go together
        with pytest.raises(_abi.TvkError):
            bad()


def test_gradient_formula():
    """Against central differences, whose error is of order step^2 and cancellation's 1e-15 / step."""
    from tests.test_distill_gpu import oracle

    g = torch.Generator().manual_seed(0)
    x = torch.randn((3, 9), generator=g, dtype=torch.float64) * 2
    index = torch.tensor([[1, 4, 1, -1], [0, 8, 3, 2], [-1, -1, -1, -1]])
    teacher, dloss = torch.randn((3, 4), generator=g, dtype=torch.float64), torch.tensor([1.0, -2.0, 3.0], dtype=torch.float64)
    step = 1e-5
    for heat in (1.0, 2.5):
        grad = oracle(x, index, teacher, heat, dloss)[1]
        for i in range(x.numel()):
            d = torch.zeros(x.numel(), dtype=torch.float64)
            d[i] = step
            up, down = ((oracle(x + s * d.view(x.shape), index, teacher, heat)[0] * dloss).sum() for s in (1, -1))
            assert abs((up - down) / (2 * step) - grad.flatten()[i]) < 1e-8
