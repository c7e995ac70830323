"""Sequences with fewer new tokens than the call: tvk_paged_append and tvk_paged_attention with new_lens, and the cache of
torchvulkan_amd.decoder that keeps them. Padding is neither written nor attended, whatever its position."""
from __future__ import annotations

import pytest
import torch

from tests.test_paged_cache_gpu import BF16, DEV, F8, HALF, Cache, attention_oracle, close, rand, rotary_table
from torchvulkan_amd import _abi, decoder

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 64), (33, 32), (80, None)])
@pytest.mark.parametrize("dtype,cache_dtype", [(HALF, HALF), (BF16, F8), (torch.float32, torch.float32)])
def test_append_leaves_padding_alone(gpu, dim, rot, dtype, cache_dtype):
    # as if every sequence's own tokens were appended by a call of their own, bit for bit
    lens, fresh, new = [30, 17, 9, 40, 5, 0, 3], [1, 17, 0, 6, 99, 4, -2], 17
    cache = Cache(lens, 16, 2, dim, cache_dtype, seed=dim)
    table = None if rot is None else rotary_table(50, rot).to(DEV)
    heads = rand((len(lens), new, 8, dim), dtype, 1).to(DEV)
    q, k, v = heads.split([4, 2, 2], 2)
    (kc, vc, dl, dt), scales = cache.dev()
    alone = kc.clone(), vc.clone()
    got = _abi.paged_append(q, k, v, kc, vc, dl, dt, rotary=table, new_lens=torch.tensor(fresh, dtype=torch.int32, device=DEV),
                            **scales)
    for b, n in enumerate(fresh):
        n = min(max(n, 0), new)
        at = slice(new - n, new)
        assert got[b, :new - n].eq(0).all()
        if n:
            want = _abi.paged_append(q[b:b + 1, at], k[b:b + 1, at], v[b:b + 1, at], *alone, dl[b:b + 1], dt[b:b + 1],
                                     rotary=table, **scales)
            assert torch.equal(got[b, at], want[0])
    for now, want in ((kc, alone[0]), (vc, alone[1])):
        assert torch.equal(now.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))


@pytest.mark.parametrize("lens,fresh,new,hq,hkv", [
    ([30, 17, 9, 40, 5], [1, 17, 0, 6, 5], 17, 4, 2), ([60, 33], [1, 0], 1, 4, 2),        # a wave each
    ([300, 500, 90, 17, 400], [1, 20, 90, 17, 0], 90, 8, 2),                               # a workgroup each
    ([3000, 40, 2222, 700], [1, 40, 0, 9], 40, 8, 2), ([9000, 5], [3, 0], 4, 8, 1),        # pieces that are joined
    ([1700 + 7 * i for i in range(40)], [i % 9 for i in range(40)], 8, 16, 8),             # many segments
])
@pytest.mark.parametrize("dim,dtype,cache_dtype", [(64, BF16, BF16), (128, BF16, F8), (64, torch.float32, torch.float32),
                                                   (40, HALF, HALF)])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_of_own_tokens(gpu, lens, fresh, new, hq, hkv, dim, dtype, cache_dtype, window):
    for page in (16, 20):
        cache = Cache(lens, page, hkv, dim, cache_dtype, seed=dim, stale=float("nan"))
        if cache_dtype != F8:
            cache.v[cache.table[0, (lens[0] - 1) // page], (lens[0] - 1) % page, 0, 3] = float("inf")   # the last token's alone
        q = rand((len(lens), new, hq, dim), dtype, 1)
        want, lse, tol = attention_oracle(q, cache, dim ** -0.5, window)
        for b, n in enumerate(fresh):
            want[b, :new - min(n, new)], lse[b, :new - min(n, new)] = 0, float("inf")
        args, scales = cache.dev()
        got, got_lse = _abi.paged_attention(q.to(DEV), *args, max_len=max(lens), window=window,
                                            new_lens=torch.tensor(fresh, dtype=torch.int32, device=DEV), **scales)
        finite = want.isfinite()
        assert torch.equal(got.cpu().double()[~finite], want[~finite])
        close(torch.where(finite, got.cpu().double(), 0.0), torch.where(finite, want, 0.0), tol.nan_to_num(0, 0, 0), f"page {page}")
        assert torch.equal(got_lse.cpu().isinf(), lse.isinf())
        # and the same bits as a call whose tokens are all new
        if all(n >= new for n in fresh):
            assert torch.equal(got, _abi.paged_attention(q.to(DEV), *args, max_len=max(lens), window=window, **scales)[0])


class Dense:
    """The keys and values of each sequence as a program means them, and attention over them in float64."""

    def __init__(self, batch, table, group):
        self.keys, self.values = [[] for _ in range(batch)], [[] for _ in range(batch)]
        self.table, self.group = table, group

    def turned(self, x, pos):
        half = self.table.shape[1] // 2
        c, s = self.table[pos, :half].double(), self.table[pos, half:].double()
        a, b = x[..., :half].double(), x[..., half:].double()
        return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)

    def add(self, b, k, v):
        self.keys[b].append(self.turned(k, len(self.keys[b])))
        self.values[b].append(v)

    def attend(self, b, q, pos):
        ks, vs = torch.stack(self.keys[b][:pos + 1]).double(), torch.stack(self.values[b][:pos + 1]).double()
        x = self.turned(q, pos).double()
        return torch.stack([torch.softmax(ks[:, h // self.group] @ x[h] / x.shape[1] ** 0.5, 0) @ vs[:, h // self.group]
                            for h in range(x.shape[0])])


# the first idles or decodes while others have prompts; every sequence's keys are read again later
STEPS = ([30, 0, 3], [1, 17, 0], [0, 1, 1], [1, 0, 1], [0, 0, 20], [1, 1, 1])


@pytest.mark.parametrize("device", ["cuda", "vulkan"])
def test_cache_of_mixed_steps(gpu, device):
    hq, hkv, dim = 4, 2, 64
    cache = decoder.PagedKVCache(3, 20, 16, hkv, dim, torch.float16, device, max_len=90)
    table = decoder.rotary_table(90, dim)
    dense = Dense(3, table, 2)
    for step, counts in enumerate(STEPS):
        new = max(counts)
        q, k, v = (rand((3, new, h, dim), HALF, 10 * step + i) for i, h in enumerate((hq, hkv, hkv)))
        cache.extend(counts)
        qr = cache.append(q.to(device), k.to(device), v.to(device), table.to(device))
        out = cache.attend(qr).cpu()
        for b, n in enumerate(counts):
            assert out[b, :new - n].eq(0).all()
            for t in range(new - n, new):
                dense.add(b, k[b, t], v[b, t])
            for t in range(new - n, new):
                want = dense.attend(b, q[b, t], len(dense.keys[b]) - new + t)
                # keys and queries rounded at ties may go either way: a step of float16 in a score of |q||k| / 8
                assert (out[b, t].double() - want).abs().max() <= 2.0 ** -7, f"step {step}, sequence {b}, token {t}"


def test_captured_step_of_other_counts(gpu):
    # one captured step of a token each; sequences that have none in a replay keep their keys
    hq, hkv, dim = 4, 2, 64
    cache = decoder.PagedKVCache(3, 20, 16, hkv, dim, torch.float16, "cuda", max_len=90)
    table = decoder.rotary_table(90, dim)
    dense = Dense(3, table, 2)
    rotary = table.cuda()
    fresh = [rand((3, 1, h, dim), HALF, 1).cuda() for h in (hq, hkv, hkv)]
    cache.extend([5, 20, 1])
    q, k, v = (rand((3, 20, h, dim), HALF, 2 + i) for i, h in enumerate((hq, hkv, hkv)))
    cache.append(None, k.cuda(), v.cuda(), rotary)
    for b, n in enumerate((5, 20, 1)):
        for t in range(20 - n, 20):
            dense.add(b, k[b, t], v[b, t])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(cache.append(*fresh, rotary), max_len=90)
    for step, counts in enumerate(([1, 1, 1], [1, 0, 1], [0, 0, 1], [1, 1, 0], [1, 1, 1])):
        q, k, v = (rand((3, 1, h, dim), HALF, 40 + 10 * step + i) for i, h in enumerate((hq, hkv, hkv)))
        for to, x in zip(fresh, (q, k, v)):
            to.copy_(x)
        cache.extend(counts)
        graph.replay()
        got = out.cpu()
        for b, n in enumerate(counts):
            if not n:
                assert got[b].eq(0).all()
                continue
            dense.add(b, k[b, 0], v[b, 0])
            want = dense.attend(b, q[b, 0], len(dense.keys[b]) - 1)
            assert (got[b, 0].double() - want).abs().max() <= 2.0 ** -7, f"replay {step}, sequence {b}"


def test_tokens_of_two_extends_in_one_append(gpu):
    cache = decoder.PagedKVCache(2, 8, 16, 1, 16, torch.float32, "cuda")
    k = rand((2, 5, 1, 16), torch.float32, 1).cuda()
    cache.extend([2, 3])
    cache.extend([3, 1])
    cache.append(None, k, k)
    for b, n in enumerate((5, 4)):
        assert torch.equal(cache.k[0, cache.table[b, 0], :n], k[b, 5 - n:])


def test_replays_past_the_captured_length(gpu):
    # a step captured without a bound follows sequences that grow past what they were at capture
    hq, hkv, dim = 4, 2, 64
    cache = decoder.PagedKVCache(2, 120, 16, hkv, dim, BF16, "cuda", max_len=900)
    rotary = decoder.rotary_table(900, dim, device="cuda")
    q, k, v = (rand((2, 1, h, dim), BF16, 1).cuda() for h in (hq, hkv, hkv))
    cache.extend([5, 30])
    prompt = rand((2, 30, hkv, dim), BF16, 2).cuda()
    cache.append(None, prompt, prompt, rotary)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(cache.append(q, k, v, rotary))
    for step in range(3):
        if step:   # many positions at once, then a token at a time again
            more = rand((2, 300, hkv, dim), BF16, 3 + step).cuda()
            cache.extend(300)
            cache.append(None, more, more, rotary)
        for t, seed in ((q, 10), (k, 20), (v, 30)):
            t.copy_(rand(t.shape, BF16, seed + step))
        cache.extend(1)
        graph.replay()
        captured = out.clone()
        assert torch.equal(captured, cache.attend(cache.append(q, k, v, rotary), max_len=900))


def test_backward_passes_end_at_the_cache(gpu):
    # (the device whose autograd the package serves)
    cache = decoder.PagedKVCache(2, 8, 16, 1, 16, torch.float32, "vulkan")
    x = rand((2, 1, 1, 16), torch.float32, 1).to("vulkan")
    leaf = x.clone().requires_grad_()
    cache.extend(1)
    for result in (lambda: cache.append(leaf * 2, x, x), lambda: cache.attend(leaf * 2), lambda: decoder.rms_norm_fp8(leaf * 2)[1]):
        with pytest.raises(_abi.TvkUnsupported):
            result().sum().backward()
    out = torch.empty_like(x)
    assert torch.equal(cache.attend(leaf).detach().cpu(), cache.attend(x, out=out).cpu())
