"""CPU checks of sampling: what its entry points refuse, and the GPU tests'
oracle against probabilities worked out by hand."""
import ctypes as C
import math

import pytest
import torch

from torchvulkan_amd import _abi, decoder

lib = _abi.load()


def desc(**kw):
    d = _abi.SampleDesc()
    d.dtype = _abi.TVK_F32
    d.rows, d.cols = 4, 100
    d.logits = d.random = d.token = 16   # never dereferenced by validation
    d.logits_stride = 100
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,want", [
    ({"dtype": _abi.TVK_F64}, "UNSUPPORTED"), ({"rows": -1}, "INVALID"), ({"cols": -1}, "INVALID"), ({"rows": 1 << 31}, "UNSUPPORTED"),
    ({"cols": (1 << 19) + 1}, "UNSUPPORTED"), ({"logits": None}, "INVALID"), ({"random": None}, "INVALID"), ({"token": None}, "INVALID"),
    ({"logits_stride": -1}, "INVALID"), ({"rows": 0}, "OK"),
])
def test_refusals(kw, want):
    st = lib.tvk_sample(C.byref(desc(**kw)))
    assert _abi.STATUS_NAMES[st] == want and (st == _abi.TVK_OK or b"tvk_sample" in lib.tvk_last_error())


def test_null_descriptor():
    assert lib.tvk_sample(None) == _abi.TVK_ERR_INVALID and b"tvk_sample" in lib.tvk_last_error()


def test_binding_refuses_other_layouts():
    x, u, t = torch.zeros((3, 50)), torch.zeros(3), torch.zeros(3, dtype=torch.int64)
    make = _abi.make_sample_desc
    make(x, u, t, u, u, t.int(), u, u)
    make(x[:1].expand(3, 50), u, t)
    for bad in (lambda: make(x[0], u, t), lambda: make(x, u[:2], t), lambda: make(x, u.double(), t), lambda: make(x, u, t.int()),
                lambda: make(x, u, t, top_k=t), lambda: make(x, u, t, top_p=t.int()), lambda: make(x, u, t, temperature=u[:1]),
                lambda: make(x.t(), u, t), lambda: make(x.double(), u, t), lambda: make(x, u, t, min_p=u.half()),
                lambda: decoder.sample(x, u), lambda: decoder.sample(x, u[:2]), lambda: decoder.sample(x, u, top_k=t),
                lambda: decoder.sample(x, u, top_p=u[:1])):
        with pytest.raises(_abi.TvkError):
            bad()


def test_oracle_by_hand():
    from tests.test_sample_gpu import oracle

    l = [math.log(v) for v in (1.0, 4.0, 2.0, 1.0, 2.0)]   # weights 1 4 2 1 2

    def drawn(u, **kw):
        return oracle(torch.tensor([l]), torch.tensor([u]), **{k: [v] for k, v in kw.items()})[0][0]

    assert [drawn(u) for u in (0.0, 0.09, 0.11, 0.49, 0.51, 0.69, 0.71, 0.79, 0.81, 0.999)] == [0, 0, 1, 1, 2, 2, 3, 3, 4, 4]
    assert [drawn(u, top_k=2) for u in (0.0, 0.6, 0.7, 0.999)] == [1, 1, 2, 2]          # the first of the twos
    assert [drawn(u, top_k=3) for u in (0.0, 0.51, 0.76)] == [1, 2, 4]
    assert [drawn(u, top_p=0.45) for u in (0.0, 0.65, 0.7)] == [1, 1, 2]
    assert [drawn(u, top_k=4, top_p=0.4) for u in (0.0, 0.99)] == [1, 1]                # 4 of 9
    assert [drawn(u, min_p=0.3) for u in (0.0, 0.51, 0.76)] == [1, 2, 4]
    assert drawn(0.7, temperature=0.0) == 1
    assert abs(oracle(torch.tensor([l]), torch.tensor([0.6]), top_k=[3])[1][0] - math.log(2 / 8)) < 1e-7
