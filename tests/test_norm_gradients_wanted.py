"""What a norm's backward call is given, on the CPU: the gradients that there are, and no zeros in place of the others."""
import pytest
import torch

from torchvulkan_amd import decoder


@pytest.fixture
def queued(monkeypatch):
    """The calls by name, none of them made."""
    calls = []
    monkeypatch.setattr(decoder, "_stream", lambda t: None)
    monkeypatch.setattr(decoder, "_queue", lambda name, desc, t: calls.append((name, desc)))
    return calls


@pytest.mark.parametrize("norm", [decoder.rms_norm, decoder.layer_norm])
@pytest.mark.parametrize("wanted", ["y", "h", "both"])
def test_with_a_residual(queued, norm, wanted):
    x, r, w = torch.zeros((3, 40), requires_grad=True), torch.zeros((3, 40), requires_grad=True), torch.ones(40, requires_grad=True)
    y, h = norm(x, w, residual=r)
    (y.sum() if wanted == "y" else h.sum() if wanted == "h" else (y + h).sum()).backward()
    assert len(queued) == 2 and queued[1][0].endswith("_norm_bwd")
    d = queued[1][1]
    assert d.dy and d.h and d.dx and d.dweight   # (a call without dy has zeros of its own)
    assert bool(d.dh) == (wanted != "y")
    assert x.grad.shape == r.grad.shape == (3, 40) and w.grad.shape == (40,)


@pytest.mark.parametrize("norm", [decoder.rms_norm, decoder.layer_norm])
def test_without_one(queued, norm):
    x = torch.zeros((3, 40), requires_grad=True)
    norm(x).sum().backward()
    assert not queued[1][1].dh and not queued[1][1].dweight and x.grad.shape == (3, 40)
