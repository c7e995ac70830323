"""A small decoder that serves a batch of prompts from a paged key/value cache:
every prompt in one call, then a token at a time, the step captured once as a HIP
graph and replayed while the sequences grow, and a training step of its norms.

    python examples/decode.py [--batch 8] [--prompt 200] [--tokens 64] [--layers 4] [--cache fp8]

Random weights and tokens: it shows the calls and their times, not language."""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from torchvulkan_amd import _abi, decoder  # noqa: E402


class Block:
    """norm, attention over the cache, norm, feed-forward: weights in [out, in] rows as nn.Linear keeps them."""

    def __init__(self, dim, heads, heads_kv, head_dim, hidden, gen, dtype, device):
        def weight(*shape):
            return (torch.randn(shape, generator=gen) / shape[-1] ** 0.5).to(dtype).to(device)

        self.heads, self.heads_kv, self.head_dim = heads, heads_kv, head_dim
        self.qkv, self.proj = weight((heads + 2 * heads_kv) * head_dim, dim), weight(dim, heads * head_dim)
        self.up, self.down = weight(hidden, dim), weight(dim, hidden)
        self.norm1, self.norm2 = (torch.ones(dim, dtype=dtype, device=device) for _ in range(2))

    def __call__(self, x, residual, cache, layer, rotary, max_len):
        b, new, dim = x.shape
        if residual is None:
            y, h = decoder.rms_norm(x, self.norm1), x
        else:
            y, h = decoder.rms_norm(x, self.norm1, residual)
        q, k, v = linear(y, self.qkv).view(b, new, -1, self.head_dim).split([self.heads, self.heads_kv, self.heads_kv], 2)
        q = cache.append(q, k, v, rotary, out=q, layer=layer)   # rotated in place
        a = cache.attend(q, max_len=max_len, layer=layer)
        y, h = decoder.rms_norm(linear(a.flatten(2), self.proj), self.norm2, h)
        return linear(linear(y, self.up, _abi.TVK_ACT_RELU), self.down), h


def linear(x, w, activation=0):
    out = torch.empty((*x.shape[:-1], w.shape[0]), dtype=x.dtype, device=x.device)
    _abi.gemm(x.reshape(-1, x.shape[-1]), w.t(), out.view(-1, w.shape[0]), activation=activation)
    return out


class Decoder:
    def __init__(self, layers=4, dim=1024, heads=16, heads_kv=4, head_dim=64, hidden=4096, vocab=4096, dtype=torch.bfloat16,
                 device="cuda", seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.blocks = [Block(dim, heads, heads_kv, head_dim, hidden, gen, dtype, device) for _ in range(layers)]
        self.embedding = torch.randn((vocab, dim), generator=gen).to(dtype).to(device)
        self.norm = torch.ones(dim, dtype=dtype, device=device)
        self.kind = dict(heads_kv=heads_kv, head_dim=head_dim, device=device)
        self.rotary = {}

    def cache(self, batch, max_len, page_size=16, dtype=torch.bfloat16):
        pages = batch * -(-max_len // page_size)
        scales = {}
        if dtype == torch.float8_e4m3fn:
            scales = {n: torch.full((self.kind["heads_kv"],), 1 / 16, device=self.kind["device"]) for n in ("k_scale", "v_scale")}
        self.table = decoder.rotary_table(max_len, self.kind["head_dim"], device=self.kind["device"])
        return decoder.PagedKVCache(batch, pages, page_size, dtype=dtype, max_len=max_len, layers=len(self.blocks), **self.kind, **scales)

    def __call__(self, tokens, cache, max_len=None):
        """Logits [batch, vocab] after the newest tokens [batch, new], whose positions the cache already has."""
        x, h = self.embedding[tokens], None
        for layer, block in enumerate(self.blocks):
            x, h = block(x, h, cache, layer, self.table, max_len)
        y, _ = decoder.rms_norm(x[:, -1:].contiguous(), self.norm, h[:, -1:].contiguous())
        return linear(y[:, 0], self.embedding)


def generate(model, prompts, count, cache_dtype=torch.bfloat16, capture=True):
    """(`count` tokens after each prompt [batch, length], greedily; seconds for the prompts; seconds a token)."""
    batch, length = prompts.shape
    cache = model.cache(batch, length + count, dtype=cache_dtype)
    cache.extend(length)
    torch.cuda.synchronize()
    begin = time.perf_counter()
    token = model(prompts, cache).argmax(-1, keepdim=True)
    torch.cuda.synchronize()
    first = time.perf_counter() - begin
    out, graph = [token.clone()], None
    if capture:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            after = model(token, cache, max_len=length + count).argmax(-1, keepdim=True)
    torch.cuda.synchronize()
    begin = time.perf_counter()
    for _ in range(count - 1):
        cache.extend(1)
        if graph:
            graph.replay()
            token.copy_(after)
        else:
            token = model(token, cache).argmax(-1, keepdim=True)
        out.append(token.clone())
    torch.cuda.synchronize()
    return torch.cat(out, 1), first, (time.perf_counter() - begin) / max(1, count - 1)


def norm_step(rows=4096, cols=1024, steps=3, rate=0.1, dtype=torch.bfloat16, device="vulkan"):
    """Fits a norm's weight to another's by gradient descent, on the device whose autograd the package serves; the losses."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randn((rows, cols), generator=gen).to(dtype).to(device)
    weight = torch.ones(cols, device=device, requires_grad=True)
    target = decoder.rms_norm(x, torch.full((cols,), 1.5, device=device)).float()
    losses = []
    for _ in range(steps):
        d = decoder.rms_norm(x, weight).float() - target
        loss = (d * d).sum() * (1 / d.numel())
        grad, = torch.autograd.grad(loss, weight)
        with torch.no_grad():
            weight -= rate * cols * grad
        losses.append(float(loss.detach()))
    return losses


def main():
    p = argparse.ArgumentParser(description=__doc__)
    p.add_argument("--batch", type=int, default=8)
    p.add_argument("--prompt", type=int, default=200)
    p.add_argument("--tokens", type=int, default=64)
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--cache", choices=["bf16", "fp8"], default="bf16")
    a = p.parse_args()
    model = Decoder(layers=a.layers)
    prompts = torch.randint(0, 4096, (a.batch, a.prompt), generator=torch.Generator().manual_seed(2)).cuda()
    dtype = torch.float8_e4m3fn if a.cache == "fp8" else torch.bfloat16
    generate(model, prompts, 4, dtype)   # builds and warms
    tokens, first, each = generate(model, prompts, a.tokens, dtype)
    print(f"{a.batch} prompts of {a.prompt}: {first * 1e3:.2f} ms; then {each * 1e6:.0f} us a token for all, "
          f"{a.batch / each:.0f} tokens/s; first tokens {tokens[0, :6].tolist()}")
    print("losses of three steps on a norm's weight:", ["%.5f" % x for x in norm_step()])


if __name__ == "__main__":
    main()
