"""tvk_paged_attention of prompts and of chunks of prompts after a cached prefix: many row blocks of two tiles' rows, keys past
what a segment takes whole, against the formula in float64 (computed on the GPU, a head and a run of tokens at a time).

Tolerances as in test_paged_cache_gpu.py, u = 2^-24 being half a float32 step: a score of D products is off by (D + 16) u of
their magnitudes' sum and its exponential by that and 2 u of the score, twice; the sums over n keys add n u of the
probability-weighted |v|; a probability rounded to a 16-bit type is off by eps / 2, and so is the output."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from torchvulkan_amd import _abi

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
HALF, BF16, F8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def rand(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


class Prompts:
    """Sequences in pages of 16 slots in a mixed order; slots without a key hold NaN."""

    def __init__(self, lens, hkv, dim, dtype, page=16, seed=0):
        need = [-(-n // page) for n in lens]
        order = torch.randperm(sum(need) + 1, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        self.table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
        self.keys, self.values, at = [], [], 0
        self.k, self.v = (torch.full((sum(need) + 1, page, hkv, dim), float("nan"), device=DEV).to(dtype) for _ in range(2))
        for b, (n, m) in enumerate(zip(lens, need)):
            self.table[b, :m] = order[at:at + m]
            at += m
            pages, slots = self.table[b].long().to(DEV), torch.arange(n, device=DEV)
            for cache, kept, s in ((self.k, self.keys, 1), (self.v, self.values, 2)):
                x = rand((n, hkv, dim), dtype, seed + 10 * b + s)
                kept.append(x)
                bits = torch.uint8 if dtype == F8 else dtype
                cache.view(bits)[pages[slots // page], slots % page] = x.view(bits)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.table = self.table.to(DEV)

    def args(self):
        return self.k, self.v, self.lens, self.table


def check(got, got_lse, q, cache, scale, window=0, step=1024):
    b, new, hq, dim = q.shape
    eps = torch.finfo(q.dtype).eps / 2
    for i in range(b):
        n = int(cache.lens[i])
        group = hq // cache.keys[i].shape[1]
        pos = torch.arange(n, device=DEV)
        for h in range(hq):
            k, v = (x[i][:, h // group].double().t().contiguous().t() for x in (cache.keys, cache.values))
            for t0 in range(0, new, step):
                x = q[i, t0:t0 + step, h].double()
                place = n - new + t0 + torch.arange(x.shape[0], device=DEV)[:, None]
                seen = (pos <= place) & (pos > place - window if window else True)
                s = torch.where(seen, (x @ k.t()) * scale, float("-inf"))
                size = torch.where(seen, (x.abs() @ k.abs().t()) * scale, 0.0).amax(-1, keepdim=True)
                top = torch.where(seen, s, 0.0).abs().amax(-1, keepdim=True)
                none = ~seen.any(-1, keepdim=True)
                p = torch.where(none, 0.0, torch.softmax(s, -1))
                want, mean = p @ v, p @ v.abs()
                err = (2 * (dim + 16) * size + 4 * top + 64 + seen.sum(-1, keepdim=True)) * U
                tol = (eps + err) * mean + eps * want.abs() + 2.0 ** -25
                out = got[i, t0:t0 + step, h].double()
                assert ((out - want).abs() <= tol).all(), f"sequence {i}, head {h}, tokens from {t0}"
                lse = got_lse[i, t0:t0 + step, h].double()[:, None]
                want = torch.where(none, float("inf"), torch.logsumexp(s, -1, keepdim=True))
                assert torch.equal(lse.isinf(), none) and ((lse - want).abs()[~none] <= 1e-4 * (1 + want.abs()[~none])).all()


# cut into chunks, into stretches, and prompts whose tokens in front of a sequence's start see nothing
@pytest.mark.parametrize("lens,hq,hkv,new,dim", [
    ([1620, 1600, 1580, 1600], 8, 4, 130, 64), ([1700, 1600], 16, 4, 350, 64), ([2500, 1700, 900, 3000], 8, 2, 700, 64),
    ([3000], 16, 8, 3000, 128), ([2000, 40, 4000], 8, 2, 2000, 128), ([6000, 5000], 4, 1, 1100, 80), ([1900] * 3, 8, 2, 513, 256),
])
@pytest.mark.parametrize("cache_dtype", ["same", F8])
@pytest.mark.parametrize("window", [0, 700])
def test_prompts(gpu, lens, hq, hkv, new, dim, cache_dtype, window):
    dtype = BF16 if dim != 80 else HALF
    cache = Prompts(lens, hkv, dim, dtype if cache_dtype == "same" else F8, seed=dim)
    q = rand((len(lens), new, hq, dim), dtype, 1)
    got, lse = _abi.paged_attention(q, *cache.args(), max_len=max(lens), window=window)
    again, lse2 = _abi.paged_attention(q, *cache.args(), max_len=max(lens), window=window)
    assert torch.equal(got, again) and torch.equal(lse, lse2)
    check(got, lse, q, cache, dim ** -0.5, window)


def test_prompt_of_more_workgroups_than_stretches(gpu):
    # a launch of 42512 workgroups, of which those with a stretch of 107749 tiles have work
    cache = Prompts([42000], 8, 128, BF16, page=64)
    q = rand((1, 42000, 32, 128), BF16, 1)
    got, lse = _abi.paged_attention(q, *cache.args(), max_len=42000)
    check(got, lse, q, cache, 128 ** -0.5, step=2000)


def reserved():
    v = C.c_size_t()
    _abi.check(_abi.load().tvk_memory_reserved(0, C.byref(v)))
    return v.value


def test_scratch_of_a_prompt(gpu):
    # partials go by the workgroups that run together: a prompt of 8192 segments takes no more than the pool's smallest buffers
    cache = Prompts([8192], 8, 128, BF16, page=64)
    q = rand((1, 8192, 32, 128), BF16, 1)
    torch.cuda.synchronize()
    _abi.check(_abi.load().tvk_empty_cache(0))
    before = reserved()
    eager, _ = _abi.paged_attention(q, *cache.args(), max_len=8192)
    assert reserved() - before <= 32 << 20
    out, graph = torch.empty_like(q), torch.cuda.CUDAGraph()
    before = reserved()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        d = _abi.make_paged_attention_desc(q, cache.k, cache.v, out, cache.lens, cache.table, max_len=8192,
                                           stream=torch.cuda.current_stream().cuda_stream)
        _abi.check(_abi.load().tvk_paged_attention(C.byref(d)))
    assert reserved() - before <= 32 << 20
    for _ in range(2):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
