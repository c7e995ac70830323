"""Backward passes of norms with a residual that come from y alone, from h alone and from both, against autograd in 64 bits.
float32 rows of 300: sums of 300 products, 2 (300 / 256 + 32) 2^-24 of their terms' magnitudes at most, a few products more: 1e-5
of the gradient's size, which stays below 20 here, is allowed."""
import pytest
import torch

from torchvulkan_amd import decoder

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("wanted", ["y", "h", "both"])
def test_with_a_residual(gpu, kind, wanted):
    g = torch.Generator().manual_seed(1)
    values = [torch.randn(s, generator=g) for s in ((5, 300), (5, 300), (300,), (300,))]
    dy, dh = torch.randn((5, 300), generator=g), torch.randn((5, 300), generator=g)
    if kind == "rms":
        values = values[:3]

    def loss(y, h, dy, dh):
        return (0 if wanted == "h" else (y * dy).sum()) + (0 if wanted == "y" else (h * dh).sum())

    dev = [t.to("vulkan").requires_grad_() for t in values]
    norm = decoder.rms_norm if kind == "rms" else decoder.layer_norm
    loss(*norm(dev[0], *dev[2:], residual=dev[1]), dy.to("vulkan"), dh.to("vulkan")).backward()
    ref = [t.double().requires_grad_() for t in values]
    h = ref[0] + ref[1]
    if kind == "rms":
        y = h / (h * h).mean(-1, keepdim=True).add(1e-5).sqrt() * ref[2]
    else:
        y = torch.nn.functional.layer_norm(h, (300,), ref[2], ref[3], 1e-5)
    loss(y, h, dy.double(), dh.double()).backward()
    for a, b in zip(dev, ref):
        want = torch.zeros_like(b) if b.grad is None else b.grad
        assert (a.grad.cpu().double() - want).abs().max().item() <= 2e-4
