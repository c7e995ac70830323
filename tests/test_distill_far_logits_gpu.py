"""The distillation loss's gradient where the logits lie far from zero: as exact as about zero.

A probability is exp((x - m) / T - log s), m the largest logit and s the sum over the row of exp((x - m) / T). With u = 2^-24 and
r = log p: the difference, its quotient, the second difference and the exponent's factor are off by u each of at most
|r| + log s, four in all and two more for the exponential and its square; s by f = 2 (cols / 256 + 64) u of itself, which
log s is off by, and by u of its own. So p is off by e = f + 6 u (|r| + 2 log(cols) + 1) of itself, and so is q, of the entries. Far
from zero float32 logits have fewer places, which is no error: they are what is given, here and in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from torchvulkan_amd import _abi, decoder

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -125, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -125}   # a p below 2^-126 is zero


def inputs(rows, cols, top, far, dtype):
    g = torch.Generator().manual_seed(cols)
    x = (torch.randn((rows, cols), generator=g) * 3 + far).to(dtype)
    index = torch.stack([torch.randperm(cols, generator=g)[:top] for _ in range(rows)])
    index[-1] = -1
    return x, index, torch.randn((rows, top), generator=g) * 2


def check(x, index, teacher, heat, got, dtype):
    rows, cols = x.shape
    logp, logq = torch.log_softmax(x.double() / heat, -1), torch.log_softmax(teacher.double() / heat, -1)
    p, there = logp.exp(), torch.zeros_like(logp)
    q = torch.where(index >= 0, logq.exp(), 0.0)
    there.scatter_add_(1, index.clamp(min=0), q)
    p[-1] = 0
    want = (p - there) * heat
    e = 2 * (cols / 256 + 64) * U + 6 * U * (logp.abs() + 2 * math.log(cols) + 1)
    tol = heat * (p + there) * e + torch.finfo(dtype).eps / 2 * want.abs() + TINY[dtype]
    assert ((got.double().cpu() - want).abs() <= tol).all()
    assert not got[-1].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("far", [0.0, 100.0, -5000.0, 30000.0])
@pytest.mark.parametrize("rows,cols,top", [(40, 500, 9), (3, 20000, 33)])
def test_gradient(gpu, dtype, far, rows, cols, top):
    x, index, teacher = inputs(rows, cols, top, far, dtype)
    for heat in (1.0, 2.0):
        leaf = x.to("vulkan").requires_grad_()
        decoder.distill_loss(leaf, index.to("vulkan"), teacher.to("vulkan"), heat).sum().backward()
        check(x, index, teacher, heat, leaf.grad, dtype)


@pytest.mark.parametrize("far", [0.0, 5000.0])
def test_calls(gpu, far):
    """The largest logit and the logarithm of the sum, beside lse or alone; dlogits over the logits."""
    x, index, teacher = inputs(12, 3000, 9, far, torch.float32)
    dev = [t.to(DEV) for t in (x, index, teacher)]
    softmax = torch.empty((12, 2), device=DEV)
    loss, lse, target = _abi.distill_fwd(*dev, softmax=softmax)
    assert torch.equal(softmax[:-1, 0], dev[0][:-1].amax(-1)) and softmax[-1, 1] == math.inf
    assert (softmax[:-1].double().sum(-1).cpu() - torch.logsumexp(x[:-1].double(), -1)).abs().max() <= 200 * U
    assert all(torch.equal(a, b) for a, b in zip(_abi.distill_fwd(*dev), (loss, lse, target)))
    one = torch.ones(12, device=DEV)
    got = _abi.distill_bwd(dev[0], dev[1], None, target, one, softmax=softmax)
    check(x, index, teacher, 1.0, got, torch.float32)
    assert torch.equal(_abi.distill_bwd(dev[0], dev[1], lse, target, one, softmax=softmax), got)
    d = _abi.make_distill_bwd_desc(dev[0], dev[1], None, target, one, dev[0], softmax=softmax, stream=torch.cuda.current_stream().cuda_stream)
    _abi.check(_abi.load().tvk_distill_bwd(_abi.C.byref(d)))
    assert torch.equal(dev[0], got)


def test_rows_that_are_not_numbers(gpu):
    """As from lse: NaN where the formulas give it, zeros in a row without entries."""
    x, index, teacher = inputs(5, 300, 4, 0.0, torch.float32)
    x[0, 3], x[1, 5], x[2], x[4, 7] = math.nan, math.inf, -math.inf, math.nan
    x[3, 9] = -math.inf
    dev = [t.to(DEV) for t in (x, index, teacher)]
    softmax = torch.empty((5, 2), device=DEV)
    _, lse, target = _abi.distill_fwd(*dev, softmax=softmax)
    one = torch.ones(5, device=DEV)
    a, b = _abi.distill_bwd(dev[0], dev[1], None, target, one, softmax=softmax), _abi.distill_bwd(dev[0], dev[1], lse, target, one)
    assert torch.equal(a.isnan(), b.isnan()) and a[:3].isnan().all() and not a[3].isnan().any() and not a[4].any()
