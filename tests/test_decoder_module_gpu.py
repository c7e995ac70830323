"""torchvulkan_amd.decoder and examples/decode.py: the norm under autograd on both devices, the cache's bookkeeping with
append and attention against dense attention, and the example's captured generation against its eager one."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

import torchvulkan_amd  # noqa: F401  (registers the vulkan device)
from torchvulkan_amd import _abi, decoder

pytestmark = pytest.mark.gpu


def rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def plain_norm(x, w, eps):
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return y if w is None else y * w


@pytest.mark.parametrize("with_residual,with_weight", [(False, True), (True, True), (True, False)])
def test_norm_under_autograd(gpu, with_residual, with_weight):
    # on the vulkan device: torch's engine follows one accelerator's streams, with it registered not cuda's
    device = "vulkan"
    # float32: a row's 200 terms, and the sums over 15 rows, are off by at most 2^-24 each of their magnitudes' sum
    x, r, w = rand(3, 5, 200, seed=1), rand(3, 5, 200, seed=2), rand(200, seed=3) + 1
    dy, dh = rand(3, 5, 200, seed=4), rand(3, 5, 200, seed=5)
    leaves = [t.to(device).requires_grad_() for t in (x, r, w)]
    ref = [t.double().requires_grad_() for t in (x, r, w)]
    if with_residual:
        y, h = decoder.rms_norm(leaves[0], leaves[2] if with_weight else None, leaves[1], eps=0.01)
        rh = ref[0] + ref[1]
        ((y * dy.to(device)).sum() + (h * dh.to(device)).sum()).backward()
        ((plain_norm(rh, ref[2] if with_weight else None, 0.01) * dy.double()).sum() + (rh * dh.double()).sum()).backward()
        assert torch.equal(h.detach().cpu(), x + r)
    else:
        y = decoder.rms_norm(leaves[0], leaves[2], eps=0.01)
        (y * dy.to(device)).sum().backward()
        (plain_norm(ref[0], ref[2], 0.01) * dy.double()).sum().backward()
    for got, want in zip(leaves, ref):
        assert (got.grad is None) == (want.grad is None)
        if want.grad is not None:
            assert ((got.grad.cpu().double() - want.grad).abs() <= 1e-4 * (want.grad.abs() + 1)).all()


@pytest.mark.parametrize("device", ["cuda", "vulkan"])
def test_norm_in_8_bits(gpu, device):
    x = rand(4, 96, dtype=torch.bfloat16)
    y, scale, h = decoder.rms_norm_fp8(x.to(device))
    want = plain_norm(x.double(), None, 1e-5)
    got = y.cpu().double() * scale.cpu().double()[:, None]
    # half a step of 8 bits, of the value or the smallest step
    assert ((got - want).abs() <= 2.0 ** -4 * 1.001 * want.abs() + 2.0 ** -10 * scale.cpu().double()[:, None]).all()
    assert h.shape == x.shape


@pytest.mark.parametrize("device", ["cuda", "vulkan"])
def test_cache_grows_like_dense_attention(gpu, device):
    hq, hkv, dim = 4, 2, 64
    cache = decoder.PagedKVCache(3, 20, 16, hkv, dim, torch.float16, device, max_len=90)
    table = decoder.rotary_table(90, dim)
    half = dim // 2
    keys, values = [[] for _ in range(3)], [[] for _ in range(3)]

    def turned(x, pos):
        c, s = table[pos, :half].double(), table[pos, half:].double()
        a, b = x[..., :half].double(), x[..., half:].double()
        return torch.cat([a * c - b * s, b * c + a * s], -1).to(torch.float16)

    for step, counts in enumerate(([17, 3, 0], [1, 1, 1], [1, 1, 1], [30, 30, 30], [1, 0, 1])):
        new = max(counts)
        q, k, v = (rand(3, new, h, dim, seed=10 * step + i, dtype=torch.float16) for i, h in enumerate((hq, hkv, hkv)))
        if step == 3:
            cache.release(1)
            keys[1], values[1] = [], []
        cache.extend(counts)
        qr = cache.append(q.to(device), k.to(device), v.to(device), table.to(device))
        out = cache.attend(qr)
        qr, out = qr.cpu(), out.cpu()
        for b, n in enumerate(counts):
            assert cache.length(b) == len(keys[b]) + n
            for t in range(new - n, new):
                pos = len(keys[b])
                keys[b].append(turned(k[b, t], pos))
                values[b].append(v[b, t])
                ks, vs = torch.stack(keys[b]).double(), torch.stack(values[b]).double()
                for h in range(hq):
                    p = torch.softmax(ks[:, h // 2] @ turned(q[b, t, h], pos).double() / dim ** 0.5, 0)
                    want = p @ vs[:, h // 2]
                    # keys and queries rounded at ties may go either way: a step of float16 in a score of |q||k| / 8
                    assert (out[b, t, h].double() - want).abs().max() <= 2.0 ** -7
    with pytest.raises(_abi.TvkError):
        cache.extend(60)
    assert [cache.length(b) for b in range(3)] == [50, 30, 33]


@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float8_e4m3fn])
def test_example_captured_and_eager(gpu, cache):
    spec = importlib.util.spec_from_file_location("decode_example", Path(__file__).resolve().parent.parent / "examples" / "decode.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    model = example.Decoder(layers=2, dim=256, heads=4, heads_kv=2, hidden=512, vocab=500)
    prompts = torch.randint(0, 500, (3, 37), generator=torch.Generator().manual_seed(0)).cuda()
    eager = example.generate(model, prompts, 12, cache, capture=False)[0]
    captured = example.generate(model, prompts, 12, cache, capture=True)[0]
    assert eager.shape == (3, 12) and torch.equal(eager[:, 0], captured[:, 0])
    # max_len deals the keys otherwise, so that a near tie of logits may fall the other way, and all after it
    assert (eager == captured).float().mean() > 0.5
    losses = example.norm_step(512, 256)
    assert losses[0] > losses[1] > losses[2]
