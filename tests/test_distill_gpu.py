"""tvk_distill_fwd / tvk_distill_bwd against the formulas in float64.

Tolerances count roundings, u = 2^-24. A row's sum of exponentials runs through
at most cols / 256 additions in a thread, an eighth as many rescalings, and the
joins: f = 2 (cols / 256 + 64) u of itself covers them with the exponentials'
own last places. An exponent (x - m) / T, x / T - lse or a logarithm of that size
is off by a few u of its terms, none above 2 A + log(cols) with A the largest
finite |x| / T or |t| / T: a = 4 u (2 A + log(cols) + 2). So log p and log q are off by
at most f + a each and p and q by as much of themselves, for both lists: e = 2 f + 2 a + 4 u."""
from __future__ import annotations

import math

import pytest
import torch

from torchvulkan_amd import _abi, decoder

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def oracle(x, index, teacher, heat, dloss=None):
    """(loss, dlogits, sum of q (|log q| + |log p|), p + q's sums at every place) in float64."""
    x, t = x.double() / heat, teacher.double() / heat
    loss, spread = torch.zeros(len(x), dtype=torch.float64), torch.zeros(len(x), dtype=torch.float64)
    grad, size = torch.zeros_like(x), torch.zeros_like(x)
    for r in range(len(x)):
        named = (index[r] >= 0) & (index[r] < x.shape[1]) & (t[r] != -math.inf)
        at = index[r][named].long()
        if not len(at):
            continue
        logp, logq = torch.log_softmax(x[r], -1), torch.log_softmax(t[r][named], -1)
        q = logq.exp()
        loss[r] = heat ** 2 * torch.where(q > 0, q * (logq - logp[at]), 0.0).sum()
        spread[r] = (q * (logq.abs() + logp[at].abs()).nan_to_num(posinf=0.0)).sum()
        there = torch.zeros_like(x[r]).index_add_(0, at, q)
        grad[r], size[r] = logp.exp() - there, logp.exp() + there
    if dloss is not None:
        grad = grad * (dloss.double() * heat)[:, None]
    return loss, grad, spread, size


def error(x, index, teacher, heat):
    tops = [t.double()[t.isfinite()].abs().max().item() for t in (x, teacher) if t.isfinite().any()]
    f = 2 * (x.shape[1] / 256 + 64) * U
    return 2 * f + 8 * U * (2 * max(tops, default=0.0) / heat + math.log(x.shape[1] + 1) + 2) + 4 * U


def close(got, ref, tol, what):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), f"{what}: NaN in other places"
    assert torch.equal(got.isinf(), ref.isinf()), f"{what}: infinities in other places"
    over = ((got - ref).abs() - tol).nan_to_num(nan=-1.0, posinf=-1.0)
    assert over.max() <= 0, f"{what}: {over.max().item():.3e} over the tolerance"


def check(x, index, teacher, heat=1.0, dloss=None, what=""):
    dloss = torch.linspace(-1, 2, len(x)) if dloss is None else dloss
    loss, grad, spread, size = oracle(x, index, teacher, heat, dloss)
    e = error(x, index, teacher, heat)
    dev = x.to(DEV), index.to(DEV), teacher.to(DEV)
    got, lse, target = _abi.distill_fwd(*dev, temperature=heat)
    dx = _abi.distill_bwd(dev[0], dev[1], lse, target, dloss.to(DEV), heat)
    torch.cuda.synchronize()
    close(got, loss, heat ** 2 * e * (1 + spread) + 4 * U * loss.abs(), what + " loss")
    tol = (dloss.double().abs() * heat)[:, None] * (size * e + 2.0 ** -126)   # a p below float32's normal range is zero
    close(dx, grad, tol + torch.finfo(x.dtype).eps / 2 * grad.abs() + TINY[x.dtype], what + " dlogits")
    return got, lse, target, dx


def inputs(rows, cols, top, dtype, seed, std=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, cols), generator=g) * std).to(dtype)
    index = torch.randint(0, cols, (rows, top), generator=g)
    return x, index, torch.randn((rows, top), generator=g) * 2


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,top", [
    (1, 1, 1), (3, 2, 5), (2, 9, 4), (5, 255, 7), (4, 1000, 64), (3, 5003, 300), (1, 40000, 8), (40, 8200, 33), (2, 70001, 2),
    (600, 700, 5), (7, 33000, 2048)])
def test_sizes(gpu, dtype, rows, cols, top):
    """From one column to lists longer than a row has columns, whose indexes stand there many times."""
    x, index, teacher = inputs(rows, cols, top, dtype, rows + cols)
    check(x, index, teacher, what="float32 teacher")
    check(x, index.to(torch.int32), teacher.to(dtype), heat=2.5, what="int32")


@pytest.mark.parametrize("top", [63, 64, 65, 257])
@pytest.mark.parametrize("rows,cols", [(3, 9000), (700, 90)])
def test_lists_about_a_wave_s(gpu, rows, cols, top):
    """Rows that one workgroup takes and rows in pieces, with lists that one wave takes and more."""
    x, index, teacher = inputs(rows, cols, top, torch.bfloat16, top)
    index[0, 3:] = -1
    index[-1, top // 2:] = index[-1, 0]
    check(x, index, teacher, 1.25)


def test_padding_and_twice(gpu):
    x, index, teacher = inputs(6, 3000, 16, torch.float32, 3)
    index[0, 5:] = -1                     # a shorter list
    index[1] = -1                         # none
    index[2, 1::2] = 3000                 # past the columns: none either
    index[3] = 17                         # one index, sixteen times
    index[4, 3], index[4, 9] = index[4, 0], index[4, 0]
    teacher[5] = -math.inf                # entries that weigh nothing
    teacher[4, 2] = -math.inf
    x[1, 7], x[5, 9] = math.nan, math.inf   # a row without entries is not looked at
    loss, lse, target, dx = check(x, index, teacher, 1.5)
    assert loss[1] == 0 and loss[5] == 0 and not dx[1].any() and not dx[5].any()
    assert not target[3, 1:].any() and abs(target[3, 0].item() - 1) <= 40 * U
    assert target[4, 3] == 0 and target[4, 9] == 0
    big = index.clone()
    big[0, 5:] = 1 << 40                  # past 32 bits, and below zero there
    big[1] = -(1 << 33)
    again = check(x, big, teacher, 1.5)
    assert all(torch.equal(a, b) for a, b in zip((loss, lse, target, dx), again))


def test_infinite_logits(gpu):
    x, index, teacher = inputs(5, 2000, 8, torch.float32, 4)
    x[0, ::3] = -math.inf                 # masked columns, none of them the teacher's
    index[0] = torch.arange(8) * 3 + 1
    x[1, 600:] = -math.inf                # whole threads and pieces without a value
    index[1] = torch.arange(8)
    x[2, index[2, 0]] = -math.inf         # the teacher's own: an infinite loss, and a gradient all the same
    x[3] = -math.inf                      # no probabilities at all
    x[4, 5] = math.inf
    loss = check(x, index, teacher, what="infinite")[0]
    assert loss[:2].isfinite().all() and loss[2] == math.inf and loss[3:].isnan().all()
    x, index, teacher = inputs(1, 9000, 4, torch.float16, 5)
    x[0, :8500] = -math.inf
    index[0] = torch.arange(4) + 8800
    check(x, index, teacher, what="a first piece without values")
    x[0, 4000] = math.nan
    assert check(x, index, teacher, what="NaN")[3].isnan().all()


def test_large_logits(gpu):
    """Logits whose exponentials leave float32, at a temperature that spreads them further."""
    x, index, teacher = inputs(4, 5000, 9, torch.float32, 6, std=300.0)
    index[:, 0] = x.argmax(-1)
    teacher[:, 0] = 30.0
    check(x, index, teacher * 20, heat=0.25, what="large")
    check(x - 5000, index, teacher, heat=7.0, what="far from zero")


def test_strides_and_in_place(gpu):
    x, index, teacher = inputs(9, 1234, 11, torch.bfloat16, 7)
    loss, lse, target, dx = check(x, index, teacher)
    wide = torch.zeros((9, 1300), dtype=torch.bfloat16, device=DEV)
    at = wide[:, 3:1237]
    at.copy_(x)
    iw, tw, qw = torch.zeros((9, 20), dtype=torch.int64, device=DEV), torch.zeros((9, 15), device=DEV), torch.zeros((9, 12), device=DEV)
    iw[:, 5:16], tw[:, 1:12] = index.to(DEV), teacher.to(DEV)
    l2, e2 = torch.zeros(9, device=DEV), torch.zeros(9, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    lib = _abi.load()
    _abi.check(lib.tvk_distill_fwd(_abi.C.byref(_abi.make_distill_desc(at, iw[:, 5:16], tw[:, 1:12], l2, e2, qw[:, :11], stream=stream))))
    assert torch.equal(l2, loss) and torch.equal(e2, lse) and torch.equal(qw[:, :11], target) and not qw[:, 11].any()
    dl = torch.linspace(-1, 2, 9).to(DEV)
    _abi.check(lib.tvk_distill_bwd(_abi.C.byref(_abi.make_distill_bwd_desc(at, iw[:, 5:16], e2, qw[:, :11], dl, at, stream=stream))))
    assert torch.equal(at, dx) and not wide[:, :3].any() and not wide[:, 1237:].any()
    one = torch.full((1,), 0.5, device=DEV)
    a, b = (_abi.distill_bwd(x.to(DEV), index.to(DEV), lse, target, d) for d in (one.expand(9), one.repeat(9)))
    assert torch.equal(a, b)
    # a loss alone, one list for all rows
    l3 = torch.zeros(9, device=DEV)
    i1, t1 = index[:1].to(DEV).expand(9, 11), teacher[:1].to(DEV).expand(9, 11)
    _abi.check(lib.tvk_distill_fwd(_abi.C.byref(_abi.make_distill_desc(x.to(DEV), i1, t1, l3, stream=stream))))
    assert torch.equal(l3, _abi.distill_fwd(x.to(DEV), i1.contiguous(), t1.contiguous())[0])


def test_nothing(gpu):
    for rows, cols, top in ((0, 10, 3), (3, 0, 2), (3, 10, 0)):
        x, i, t = torch.zeros((rows, cols), device=DEV), torch.zeros((rows, top), dtype=torch.int64, device=DEV), torch.zeros((rows, top), device=DEV)
        loss, lse, target = _abi.distill_fwd(x, i, t)
        dx = _abi.distill_bwd(x, i, lse, target, loss)
        assert loss.shape == (rows,) and not loss.any() and not dx.any()


def test_captured(gpu):
    """Replays of a captured step, with eager calls between them, give the eager call's bits (the row cut into pieces)."""
    x, index, teacher = (t.to(DEV) for t in inputs(2, 60000, 20, torch.float32, 8))
    dl = torch.ones(2, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _abi.distill_fwd(x, index, teacher)
        dx = _abi.distill_bwd(x, index, out[1], out[2], dl)
    for i in range(3):
        x.copy_(inputs(2, 60000, 20, torch.float32, 20 + i)[0])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*out, dx)]
        want = _abi.distill_fwd(x, index, teacher)
        want = [*want, _abi.distill_bwd(x, index, want[1], want[2], dl)]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_autograd(gpu):
    """decoder.distill_loss on the vulkan device, through a mean whose gradient is one number for all rows."""
    x, index, teacher = inputs(6, 500, 9, torch.float32, 9)
    leaf = x.view(2, 3, 500).to("vulkan").requires_grad_()
    loss = decoder.distill_loss(leaf, index.view(2, 3, 9).to("vulkan"), teacher.view(2, 3, 9).to("vulkan"), 2.0)
    assert loss.shape == (2, 3)
    loss.mean().backward()
    ref, grad, spread, size = oracle(x, index, teacher, 2.0, torch.full((6,), 1 / 6))
    e = error(x, index, teacher, 2.0)
    close(loss.detach().cpu().view(6), ref, 4 * e * (1 + spread) + 4 * U * ref.abs(), "loss")
    close(leaf.grad.cpu().view(6, 500), grad, size / 3 * (e + 2 * U) + 2 * U * grad.abs(), "gradient")
