"""tvk_sample against sorting in float64.

Tokens have to be equal. The weights are integers of 2^-44, from an exponential
within 2^-46: their sums are within cols / 2 of those units of the exact ones, a
share of 2^-26 at the very most and about 2^-36 where the errors are like random
numbers, so a border or a draw falls elsewhere once in a billion. logprob is a
difference of logits over T and a logarithm in 64 bits, rounded once: half a
float32 step and what the total is off by."""
from __future__ import annotations

import math

import pytest
import torch

from torchvulkan_amd import _abi, decoder

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def oracle(x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """(tokens, logprobs) of rows, from the definition."""
    tokens, logprobs = [], []
    for r in range(len(x)):
        l = x[r].double()
        l = torch.where(l.isnan(), -math.inf, l)
        heat = float(temperature[r]) if temperature is not None else 1.0
        k = int(top_k[r]) if top_k is not None else 0
        p = float(top_p[r]) if top_p is not None else 1.0
        least = float(min_p[r]) if min_p is not None else 0.0
        top = l.max()
        if top == -math.inf:
            tokens.append(-1)
            logprobs.append(math.nan)
            continue
        w = torch.where(l == top, 1.0, torch.exp((l - top) / heat)) if heat > 0 else (l == top).double()
        w = torch.where(l == -math.inf, 0.0, w)
        order = torch.sort(l, descending=True, stable=True).indices
        if not heat > 0:
            order = order[:1]
        if k > 0:
            order = order[:k]
        if p < 1:
            sums = torch.cumsum(w[order], 0)
            order = order[:1 + int((sums < p * sums[-1]).sum())] if p > 0 else order[:1]
        if least > 0:
            order = order[w[order] >= min(least, 1.0)]
        kept = torch.sort(order).values
        sums = torch.cumsum(w[kept], 0)
        number = min(max(float(u[r]), 0.0), 1.0) if u[r] == u[r] else 0.0
        i = int((sums <= number * sums[-1]).sum())
        if i >= len(kept):   # the last that weighs anything
            i = int(w[kept].nonzero()[-1])
        tokens.append(int(kept[i]))
        logprobs.append(float(torch.log(w[kept[i]] / sums[-1])))
    return tokens, logprobs


def check(x, u, what="", **kw):
    kinds = {"top_k": torch.int32}
    dev = {name: torch.as_tensor(v).to(kinds.get(name, torch.float32)).to(DEV) for name, v in kw.items()}
    token, logprob = _abi.sample(x.to(DEV), u.to(DEV), **dev)
    torch.cuda.synchronize()
    tokens, logprobs = oracle(x, u, **{name: v.cpu() for name, v in dev.items()})
    assert token.tolist() == tokens, what
    ref = torch.tensor(logprobs, dtype=torch.float64)
    got = logprob.cpu().double()
    assert torch.equal(got.isnan(), ref.isnan()), what
    assert ((got - ref).abs() <= 2.0 ** -23 * ref.abs() + 2.0 ** -26).logical_or(ref.isnan()).all(), what
    return token, logprob


def rand(rows, cols, dtype, seed, std=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, cols), generator=g) * std).to(dtype), torch.rand(rows, generator=g)


SIZES = [(1, 1), (3, 2), (4, 7), (9, 100), (5, 513), (4, 1000), (3, 8193), (2, 50001), (1, 160003)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_filters(gpu, dtype, rows, cols):
    x, u = rand(rows, cols, dtype, rows + cols)
    heat = torch.linspace(0.3, 1.6, rows)
    check(x, u, "bare")
    check(x, u, "temperature", temperature=heat)
    for k in (1, 2, 5, 40, 300, 700, cols - 1, cols, cols + 5):
        check(x, u, f"top_k {k}", top_k=[k] * rows, temperature=heat)
    for p in (0.0, 1e-6, 0.1, 0.5, 0.9, 0.999, 1.0):
        check(x, u, f"top_p {p}", top_p=[p] * rows)
    for m in (1e-6, 0.02, 0.3, 1.0, 2.0):
        check(x, u, f"min_p {m}", min_p=[m] * rows)
    check(x, u, "together", temperature=heat, top_k=[50] * rows, top_p=[0.8] * rows, min_p=[0.01] * rows)
    check(x, u, "far in", temperature=heat, top_k=[max(1, cols // 2)] * rows, top_p=[0.97] * rows)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_of_unlike_kind(gpu, dtype):
    rows = 300
    x, u = rand(rows, 3001, dtype, 1)
    g = torch.Generator().manual_seed(2)
    pick = lambda values: torch.tensor(values)[torch.randint(0, len(values), (rows,), generator=g)]  # noqa: E731
    check(x, u, temperature=pick([0.0, 0.5, 1.0, 2.0, -1.0, math.nan]), top_k=pick([0, 1, 7, 50, 1000, 5000, -3]),
          top_p=pick([1.0, 0.9, 0.5, 0.0, 2.0, -1.0, math.nan]), min_p=pick([0.0, 0.05, 0.5, -1.0, math.nan]))


def test_equal_logits(gpu):
    """Ties go to the lowest index: at a border among hundreds of them, and in rows that are nothing else."""
    x, u = rand(6, 5000, torch.float32, 3)
    x = (x * 2).round() / 2
    for k in (1, 3, 100, 1000, 2500, 4990):
        check(x, u, f"{k}", top_k=[k] * 6)
    for p in (0.01, 0.3, 0.7, 0.95, 0.9999):
        check(x, u, f"{p}", top_p=[p] * 6, temperature=[3.0] * 6)
    same = torch.full((6, 5000), -2.5)
    same[3, 100:] = -math.inf
    for kw in ({}, {"top_k": [7] * 6}, {"top_p": [0.5] * 6}, {"top_k": [1000] * 6, "top_p": [0.251] * 6}, {"min_p": [1.0] * 6}):
        check(same, u, f"{kw}", **kw)
    signs = torch.zeros((2, 40))
    signs[:, ::2] = -0.0   # zeros of either sign are equal
    check(signs, u[:2], top_k=[5, 5])


def test_unlike_scales(gpu):
    """Values that no single histogram spreads: outliers, tight clusters, every binade."""
    u = torch.linspace(0, 0.999, 8)
    x = torch.empty((8, 4000))
    g = torch.Generator().manual_seed(5)
    x[0] = torch.randn(4000, generator=g) * 1e-6
    x[1] = torch.randn(4000, generator=g) * 1e-6 + 50
    x[2] = torch.randn(4000, generator=g) * 1e30
    x[3] = torch.ldexp(torch.ones(4000), torch.randint(-140, 4, (4000,), generator=g))
    x[4] = torch.randn(4000, generator=g)
    x[4, 17] = 3e38
    x[4, 18] = -3e38
    x[5] = torch.arange(4000) * 1e-3
    x[6] = -torch.arange(4000).float()
    x[7] = torch.nextafter(torch.ones(4000), torch.full((4000,), 2.0))
    x[7, ::3] = 1.0
    for heat in (1.0, 1e-3, 1e3, 1e38, math.inf, 1e-38):
        for kw in ({}, {"top_k": [900] * 8}, {"top_k": [3990] * 8}, {"top_p": [0.6] * 8}, {"top_k": [2000] * 8, "top_p": [0.9] * 8}):
            check(x, u, f"{heat} {kw}", temperature=[heat] * 8, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(2, 128000), (12, 70001)])
def test_borders_among_many(gpu, dtype, rows, cols):
    """Flat distributions: the border lies among hundreds or thousands of tokens of nearly one weight, much is above it."""
    for std in (0.01, 0.2, 1.0, 3.0):
        x, u = rand(rows, cols, dtype, 11, std)
        heat = torch.linspace(0.6, 2.5, rows)
        for p in (0.05, 0.5, 0.95):
            check(x, u, f"{std} {p}", top_p=[p] * rows, temperature=heat)
        check(x, u, f"{std} top_k", top_k=[cols // 3] * rows, temperature=heat)
        check(x, u, f"{std} min_p", top_p=[0.9] * rows, min_p=[0.2] * rows)


def test_masks_and_not_numbers(gpu):
    x, u = rand(9, 2000, torch.float32, 6)
    x[0] = -math.inf                       # nothing
    x[1] = math.nan
    x[2, 1:] = -math.inf                   # a single one
    x[3, :1999] = -math.inf                # the last
    x[4, ::2] = math.nan
    x[5, 100], x[5, 900], x[5, 1500] = math.inf, math.inf, math.inf
    x[6, torch.arange(2000) % 97 != 5] = -math.inf
    x[7] = torch.finfo(torch.float32).min  # the type's lowest value is a logit like others
    x[8, 50:] = torch.finfo(torch.float32).min
    for kw in ({}, {"top_k": [2] * 9}, {"top_k": [500] * 9}, {"top_p": [0.7] * 9}, {"min_p": [0.2] * 9}, {"temperature": [0.0] * 9},
               {"top_k": [30] * 9, "top_p": [0.6] * 9, "min_p": [0.01] * 9}):
        token, logprob = check(x, u, f"{kw}", **kw)
        assert token[0] == -1 and token[1] == -1 and token[2] == 0 and token[3] == 1999 and logprob[2] == 0


def test_numbers_at_the_ends(gpu):
    x, _ = rand(6, 700, torch.float32, 7)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 1.5, -0.5, math.nan])
    for kw in ({}, {"top_k": [9] * 6}, {"top_p": [0.5] * 6}):
        check(x, u, f"{kw}", **kw)


def test_every_share_of_a_row(gpu):
    """A row drawn from 4096 times at even steps: each token as often as it weighs, to one draw."""
    x, _ = rand(1, 300, torch.float32, 8)
    u = (torch.arange(4096) + 0.5) / 4096
    token, _ = _abi.sample(x.to(DEV).expand(4096, 300), u.to(DEV), top_k=torch.full((4096,), 40, dtype=torch.int32, device=DEV))
    seen = torch.bincount(token.cpu(), minlength=300)
    order = torch.sort(x[0], descending=True, stable=True).indices[:40]
    w = torch.zeros(300, dtype=torch.float64)
    w[order] = torch.softmax(x[0, order].double(), 0)
    assert ((seen - 4096 * w).abs() <= 1 + 1e-9).all() and not seen[w == 0].any()


def test_strides(gpu):
    wide, u = rand(7, 1200, torch.bfloat16, 9)
    x = wide[:, 5:1106]
    token, logprob = check(x.contiguous(), u, top_p=[0.9] * 7)
    got = _abi.sample(wide.to(DEV)[:, 5:1106], u.to(DEV), top_p=torch.full((7,), 0.9, device=DEV))
    assert torch.equal(got[0], token) and torch.equal(got[1], logprob)
    assert _abi.sample(torch.zeros((0, 9), device=DEV), torch.zeros(0, device=DEV))[0].shape == (0,)
    assert _abi.sample(torch.zeros((2, 0), device=DEV), torch.zeros(2, device=DEV))[0].tolist() == [-1, -1]


def test_captured(gpu):
    """Replays follow logits, numbers and filters that changed since, with eager calls between them."""
    x, u = (t.to(DEV) for t in rand(5, 30000, torch.bfloat16, 10))
    heat, k, p = torch.ones(5, device=DEV), torch.full((5,), 50, dtype=torch.int32, device=DEV), torch.full((5,), 0.9, device=DEV)
    _abi.sample(x, u, heat, k, p)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _abi.sample(x, u, heat, k, p)
    for i in range(3):
        nx, nu = rand(5, 30000, torch.bfloat16, 20 + i)
        x.copy_(nx)
        u.copy_(nu)
        heat.fill_(0.5 + i)
        k.fill_([7, 0, 20000][i])
        p.fill_([0.5, 0.99, 1.0][i])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, _abi.sample(x, u, heat, k, p)))


@pytest.mark.parametrize("device", ["cuda", "vulkan"])
def test_module(gpu, device):
    """decoder.sample takes numbers or tensors of the rows, in the logits' shape."""
    x, u = rand(6, 400, torch.float32, 11)
    want = oracle(x, u, [0.7] * 6, [30] * 6, [0.8] * 6, [0.02] * 6)[0]
    args = x.view(2, 3, 400).to(device), u.view(2, 3).to(device)
    token, logprob = decoder.sample(*args, 0.7, 30, 0.8, 0.02)
    assert token.shape == (2, 3) and logprob.shape == (2, 3) and token.flatten().tolist() == want
    full = lambda v, dtype=torch.float32: torch.full((2, 3), v, dtype=dtype).to(device)  # noqa: E731
    again = decoder.sample(*args, full(0.7), full(30, torch.int32), full(0.8), full(0.02))
    assert torch.equal(again[0].cpu(), token.cpu()) and torch.equal(again[1].cpu(), logprob.cpu())
    assert decoder.sample(*args, temperature=0.0)[0].flatten().tolist() == x.argmax(-1).tolist()
    if device == "vulkan":
        with pytest.raises(_abi.TvkUnsupported):
            decoder.sample(args[0].requires_grad_(), args[1])[1].sum().backward()
