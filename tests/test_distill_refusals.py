"""CPU checks of what the distillation loss refuses: temperatures beside which an exponent's factor leaves float32, and the
largest logits and sums of other shapes."""
import ctypes as C

import pytest
import torch

from tests.test_distill import filled, status
from torchvulkan_amd import _abi


@pytest.mark.parametrize("temperature", [2.95e-39, 3.5e-39, 4.2e-39])
def test_temperatures(temperature):
    """1 / T is finite in float32, log2(e) / T is not."""
    assert status("tvk_distill_fwd", filled(_abi.DistillDesc, {"temperature": temperature})) == "INVALID"
    assert status("tvk_distill_bwd", filled(_abi.DistillBwdDesc, {"temperature": temperature})) == "INVALID"


def test_softmax():
    x, i, t = torch.zeros((3, 50)), torch.zeros((3, 4), dtype=torch.int64), torch.zeros((3, 4))
    v, q, s = torch.zeros(3), torch.zeros((3, 4)), torch.zeros((3, 2))
    assert _abi.make_distill_desc(x, i, t, v, None, q, softmax=s).softmax == s.data_ptr()
    d = _abi.make_distill_bwd_desc(x, i, None, q, v, x, softmax=s)
    assert d.softmax == s.data_ptr() and not d.lse
    for bad in (v, s[:2], s.double(), torch.zeros((2, 3)).t(), torch.zeros((3, 4))[:, :2]):
        with pytest.raises(_abi.TvkError):
            _abi.make_distill_desc(x, i, t, v, softmax=bad)
        with pytest.raises(_abi.TvkError):
            _abi.make_distill_bwd_desc(x, i, v, q, v, x, softmax=bad)
    neither = _abi.make_distill_bwd_desc(x, i, None, q, v, x)
    assert _abi.load().tvk_distill_bwd(C.byref(neither)) == _abi.TVK_ERR_INVALID
