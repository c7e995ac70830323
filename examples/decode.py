"""A small decoder that serves a batch of prompts from a paged key/value cache:
every prompt in one call, then a token at a time, the step captured once as a HIP
graph and replayed while the sequences grow, and training steps of its norms and of a
head that learns from a teacher's top logits. With --weights fp8 the blocks have layer
norms that write 8 bits and products of 8-bit blocks; with --temperature (and --top-k,
--top-p, --min-p) the tokens are drawn, not the likeliest.

    python examples/decode.py [--batch 8] [--prompt 200] [--tokens 64] [--layers 4] [--cache fp8] [--weights fp8] [--temperature 0.8]

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


class Block8(Block):
    """The same with layer norms whose results are the next product's 8-bit operand, and weights in blocks of 128 x 128."""

    def __init__(self, dim, *sizes):
        super().__init__(dim, *sizes)
        self.bias1, self.bias2 = torch.zeros_like(self.norm1), torch.zeros_like(self.norm2)
        self.qkv, self.proj, self.up, self.down = (decoder.quantize_fp8(w, 128) for w in (self.qkv, self.proj, self.up, self.down))

    def __call__(self, x, residual, cache, layer, rotary, max_len):
        b, new, dim = x.shape
        y, scale, h = decoder.layer_norm_fp8(x, self.norm1, self.bias1, residual)
        qkv = decoder.linear_fp8(y, *self.qkv, x_scale=scale, out_dtype=x.dtype)
        q, k, v = qkv.view(b, new, -1, self.head_dim).split([self.heads, self.heads_kv, self.heads_kv], 2)
        q = cache.append(q, k, v, rotary, out=q, layer=layer)
        a = cache.attend(q, max_len=max_len, layer=layer)
        y, scale, h = decoder.layer_norm_fp8(decoder.linear_fp8(a.flatten(2), *self.proj), self.norm2, self.bias2, h)
        up = decoder.linear_fp8(y, *self.up, x_scale=scale, out_dtype=x.dtype)
        return decoder.linear_fp8(up.relu_(), *self.down), h


def linear(x, w, activation=0):
    out = torch.empty((*x.shape[:-1], w.shape[0]), dtype=x.dtype, device=x.device)
    _abi.gemm(x.reshape(-1, x.shape[-1]), w.t(), out.view(-1, w.shape[0]), activation=activation)
    return out


class Decoder:
    def __init__(self, layers=4, dim=1024, heads=16, heads_kv=4, head_dim=64, hidden=4096, vocab=4096, dtype=torch.bfloat16,
                 device="cuda", seed=0, block=Block):
        gen = torch.Generator().manual_seed(seed)
        self.blocks = [block(dim, heads, heads_kv, head_dim, hidden, gen, dtype, device) for _ in range(layers)]
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


def generate(model, prompts, count, cache_dtype=torch.bfloat16, capture=True, draw=None, seed=3):
    """(`count` tokens after each prompt [batch, length], the likeliest or drawn with decoder.sample's arguments `draw`; seconds
    for the prompts; seconds a token)."""
    batch, length = prompts.shape
    numbers = torch.rand((count, batch), generator=torch.Generator().manual_seed(seed)).to(prompts.device)
    number = numbers[0].clone()   # the step's, for all sequences

    def pick(logits):
        return logits.argmax(-1, keepdim=True) if draw is None else decoder.sample(logits, number, **draw)[0][:, None]

    cache = model.cache(batch, length + count, dtype=cache_dtype)
    cache.extend(length)
    torch.cuda.synchronize()
    begin = time.perf_counter()
    token = pick(model(prompts, cache))
    torch.cuda.synchronize()
    first = time.perf_counter() - begin
    out, graph = [token.clone()], None
    if capture:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            after = pick(model(token, cache, max_len=length + count))
    torch.cuda.synchronize()
    begin = time.perf_counter()
    for step in range(1, count):
        cache.extend(1)
        number.copy_(numbers[step])
        if graph:
            graph.replay()
            token.copy_(after)
        else:
            token = pick(model(token, cache))
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


class Head:
    """A layer norm and a product that learn a teacher's distribution of the next token from its largest logits."""

    def __init__(self, dim, vocab, dtype=torch.bfloat16, device="vulkan", seed=4):
        gen = torch.Generator().manual_seed(seed)
        self.product = (torch.randn((vocab, dim), generator=gen) / dim ** 0.5).to(dtype).to(device).requires_grad_()
        self.weight = torch.ones(dim, device=device, requires_grad=True)
        self.bias = torch.zeros(dim, device=device, requires_grad=True)

    def step(self, x, index, teacher, temperature=2.0, rate=0.5):
        """(loss, gradients of product, weight and bias) of a step of gradient descent: x [rows, dim], index, teacher [rows, top]."""
        leaves = [self.product, self.weight, self.bias]
        logits = torch.nn.functional.linear(decoder.layer_norm(x, self.weight, self.bias), self.product)
        loss = decoder.distill_loss(logits, index, teacher, temperature).sum() * (1 / x.shape[0])
        grads = torch.autograd.grad(loss, leaves)
        with torch.no_grad():
            for leaf, grad in zip(leaves, grads):
                leaf -= rate * grad
        return float(loss.detach()), grads


def distill_steps(rows=2048, dim=512, vocab=4096, top=64, steps=3):
    """The losses of a head's steps against a teacher that is another product of the same rows."""
    gen = torch.Generator().manual_seed(5)
    x = torch.randn((rows, dim), generator=gen).bfloat16()
    teacher, index = torch.topk(x.float() @ torch.randn((dim, vocab), generator=gen) * (2 / dim ** 0.5), top)
    head = Head(dim, vocab)
    x, index, teacher = (t.to("vulkan") for t in (x, index, teacher))
    return [head.step(x, index, teacher)[0] for _ in range(steps)]


def main():
    p = argparse.ArgumentParser(description=__doc__)
    p.add_argument("--batch", type=int, default=8)
    p.add_argument("--prompt", type=int, default=200)
    p.add_argument("--tokens", type=int, default=64)
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--cache", choices=["bf16", "fp8"], default="bf16")
    p.add_argument("--weights", choices=["bf16", "fp8"], default="bf16")
    p.add_argument("--temperature", type=float, help="draw the tokens")
    p.add_argument("--top-k", type=int, default=0)
    p.add_argument("--top-p", type=float, default=1.0)
    p.add_argument("--min-p", type=float, default=0.0)
    a = p.parse_args()
    model = Decoder(layers=a.layers, block=Block8 if a.weights == "fp8" else Block)
    draw = None if a.temperature is None else dict(temperature=a.temperature, top_k=a.top_k, top_p=a.top_p, min_p=a.min_p)
    prompts = torch.randint(0, 4096, (a.batch, a.prompt), generator=torch.Generator().manual_seed(2)).cuda()
    dtype = torch.float8_e4m3fn if a.cache == "fp8" else torch.bfloat16
    generate(model, prompts, 4, dtype, draw=draw)   # builds and warms
    tokens, first, each = generate(model, prompts, a.tokens, dtype, draw=draw)
    print(f"{a.batch} prompts of {a.prompt}: {first * 1e3:.2f} ms; then {each * 1e6:.0f} us a token for all, "
          f"{a.batch / each:.0f} tokens/s; first tokens {tokens[0, :6].tolist()}")
    print("losses of three steps on a norm's weight:", ["%.5f" % x for x in norm_step()])
    print("losses of three steps of a head against a teacher:", ["%.4f" % x for x in distill_steps()])


if __name__ == "__main__":
    main()
