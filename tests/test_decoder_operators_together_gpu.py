"""Layer norms in 8 bits, products of 8-bit blocks, the loss against a teacher and the drawing of tokens, one behind the
other as examples/decode.py uses them.

The run of a block against 64 bits: each 8-bit rounding is off by at most half a step, 2^-4 of the value (of the block's
largest / 448 times 2^-10 for the smallest). As a vector of many values whose errors are unlike, what is left of two
operands is below sqrt(2) 2^-4 = 0.089 of the product, of two products in a row below 0.13; the bfloat16 roundings between
them add 2^-8 each. Both bounds are of the relative distance of whole tensors."""
from __future__ import annotations

import ctypes as C
import importlib.util
from pathlib import Path

import pytest
import torch

from torchvulkan_amd import _abi, decoder

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("decode_example", Path(__file__).resolve().parent.parent / "examples" / "decode.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def apart(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("rows", [1, 3, 17, 200])
def test_norm_product_norm_product(gpu, rows):
    gen = torch.Generator().manual_seed(rows)
    x, r = (torch.randn((rows, 520), generator=gen).bfloat16() for _ in range(2))
    w, b = torch.rand(520, generator=gen) + 0.5, torch.randn(520, generator=gen) / 4
    up, down = torch.randn((1032, 520), generator=gen).bfloat16() / 16, torch.randn((520, 1032), generator=gen).bfloat16() / 16
    dev = [t.cuda() for t in (x, r, w, b, up, down)]
    eights = [decoder.quantize_fp8(t, 128) for t in dev[4:]]

    def block(x, r, w, b):
        y, scale, h = decoder.layer_norm_fp8(x, w, b, r)
        u = decoder.linear_fp8(y, *eights[0], x_scale=scale)
        return u, decoder.linear_fp8(u.relu(), *eights[1]), h

    u, out, h = block(*dev[:4])
    hd = x.double() + r.double()
    y = torch.nn.functional.layer_norm(hd, (520,), w.double(), b.double(), 1e-5)
    ud = y @ up.double().t()
    assert apart(h, hd) < 2.0 ** -8
    assert apart(u, ud) < 0.09 + 2.0 ** -8
    assert apart(out, ud.relu() @ down.double().t()) < 0.13 + 2.0 ** -6
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = block(*dev[:4])
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(again, (u, out, h)))
        eager = block(*dev[:4])
        assert all(torch.equal(p, q) for p, q in zip(eager, (u, out, h)))


def calls(seed):
    """Inputs of calls that take the library's scratch, and the calls: sums of a split K, rows cut among workgroups, pieces."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((130, 2100), generator=gen).bfloat16().cuda()
    w = decoder.quantize_fp8(torch.randn((400, 2100), generator=gen).bfloat16().cuda(), 128)
    logits, number = torch.randn((3, 70000), generator=gen).cuda(), torch.rand(3, generator=gen).cuda()
    index, teacher = torch.randint(0, 70000, (3, 20), generator=gen).cuda(), torch.randn((3, 20), generator=gen).cuda()
    inputs = x, logits, number, teacher

    def run():
        return (decoder.linear_fp8(x, *w), *decoder.sample(logits, number, top_p=0.9), *decoder.sample(logits, number, 0.7, 50, 0.9),
                decoder.distill_loss(logits, index, teacher, 2.0))
    return inputs, run


def test_streams_at_once(gpu):
    """The same calls on two streams: each has scratch of its own."""
    many = [calls(seed)[1] for seed in (1, 2)]
    want = [run() for run in many]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(many[k]())
    torch.cuda.synchronize()
    for k in range(2):
        for results in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(results, want[k]))


def test_two_graphs(gpu):
    """Captured one after the other, replayed in turn and beside each other with inputs that change, eager calls between them."""
    made = [calls(seed) for seed in (3, 4)]
    graphs, outs = [], []
    for _, run in made:
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(3):
        for inputs, _ in made:
            for t in inputs:
                t.copy_(t.roll(1, -1))
        want = [run() for _, run in made]
        torch.cuda.synchronize()
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], want[k]))


@pytest.mark.parametrize("draw", [None, dict(temperature=0.9, top_k=40, top_p=0.9), dict(temperature=1.3, min_p=0.02)])
def test_captured_tokens_are_the_eager_ones(gpu, example, draw):
    model = example.Decoder(layers=2, dim=256, heads=4, heads_kv=2, hidden=520, vocab=500, block=example.Block8)
    prompts = torch.randint(0, 500, (3, 70), generator=torch.Generator().manual_seed(0)).cuda()
    captured = example.generate(model, prompts, 12, draw=draw, seed=3)[0]
    assert captured.shape == (3, 12) and captured.min() >= 0 and captured.max() < 500
    numbers = torch.rand((12, 3), generator=torch.Generator().manual_seed(3)).cuda()
    cache = model.cache(3, 82)
    cache.extend(70)
    token, eager = prompts, []
    for step in range(12):
        if step:
            cache.extend(1)
        logits = model(token, cache, max_len=82 if step else None)
        token = logits.argmax(-1, keepdim=True) if draw is None else decoder.sample(logits, numbers[step], **draw)[0][:, None]
        eager.append(token)
    assert torch.equal(captured, torch.cat(eager, 1))


def test_gradients_of_a_step(gpu, example):
    """Against autograd in 64 bits. What bfloat16 leaves: the norm's rounding, 2^-8 of a value at most, is 2^-8 sum |y w| / T <=
    2^-8 * 11 / 2 = 0.021 in an exponent, the logits' 2^-8 * 5 / 2 = 0.01; so p is off by at most 0.032 of itself, p being
    the smaller part of p - q; that is rounded once, 2^-8, and so are the product's gradient and the norm's incoming one."""
    rows, dim, vocab, top = 300, 256, 1000, 16
    gen = torch.Generator().manual_seed(1)
    x = torch.randn((rows, dim), generator=gen).bfloat16()
    index = torch.stack([torch.randperm(vocab, generator=gen)[:top] for _ in range(rows)])
    teacher = torch.randn((rows, top), generator=gen) * 2
    head = example.Head(dim, vocab)
    leaves = [t.detach().cpu().double().requires_grad_() for t in (head.product, head.weight, head.bias)]
    logits = torch.nn.functional.layer_norm(x.double(), (dim,), leaves[1], leaves[2], 1e-5) @ leaves[0].t()
    q = torch.softmax(teacher.double() / 2, -1)
    lp = torch.log_softmax(logits / 2, -1).gather(1, index)
    loss = ((q * (q.log() - lp)).sum(-1) * 4).mean()
    loss.backward()
    got, grads = head.step(x.to("vulkan"), index.to("vulkan"), teacher.to("vulkan"))
    assert abs(got - float(loss.detach())) < 0.032 * 4
    for g, leaf in zip(grads, leaves):
        assert apart(g, leaf.grad) < 0.032 + 3 * 2.0 ** -8
    assert not torch.equal(head.bias.detach().cpu(), torch.zeros(dim))


def test_the_example_s_steps_run(gpu, example):
    losses = example.distill_steps(300, 128, 500, 16, 2)
    assert len(losses) == 2 and all(x == x and x > 0 for x in losses)


def test_rows_far_apart(gpu):
    """Rows 2.2 GB from each other, read and written: the bits of rows side by side."""
    apart, cols = 1_100_000_000, 3000
    stream = torch.cuda.current_stream().cuda_stream
    lib = _abi.load()
    memory = [torch.empty(2 * apart + cols, dtype=torch.bfloat16, device="cuda") for _ in range(2)]

    def far(t, where):
        out = memory[where].as_strided(t.shape, (apart, 1))
        out.copy_(t)
        return out

    gen = torch.Generator().manual_seed(6)
    x = torch.randn((3, cols), generator=gen).bfloat16().cuda()
    dy = torch.randn((3, cols), generator=gen).bfloat16().cuda()
    number = torch.rand(3, generator=gen).cuda()
    index, teacher = torch.randint(0, cols, (3, 9), generator=gen).cuda(), torch.randn((3, 9), generator=gen).cuda()
    heat = torch.full((3,), 0.9, device="cuda")
    want = _abi.sample(x, number, top_p=heat)
    assert all(torch.equal(a, b) for a, b in zip(_abi.sample(far(x, 0), number, top_p=heat), want))

    loss, lse, target = _abi.distill_fwd(x, index, teacher)
    want = _abi.distill_bwd(x, index, lse, target, number)
    xf, out = far(x, 0), far(torch.zeros_like(x), 1)
    assert all(torch.equal(a, b) for a, b in zip(_abi.distill_fwd(xf, index, teacher), (loss, lse, target)))
    _abi.check(lib.tvk_distill_bwd(C.byref(_abi.make_distill_bwd_desc(xf, index, lse, target, number, out, 1.0, stream))))
    assert torch.equal(out, want)

    want = _abi.layer_norm_fwd(x)[0]
    _abi.check(lib.tvk_layer_norm_fwd(C.byref(_abi.make_layer_norm_desc(xf, None, None, out, stream=stream))))
    assert torch.equal(out, want)
    want = _abi.layer_norm_bwd(dy, x)[0]
    dyf = far(dy, 1)   # and dx over it
    _abi.check(lib.tvk_layer_norm_bwd(C.byref(_abi.make_layer_norm_bwd_desc(dyf, far(x, 0), None, dyf, stream=stream))))
    assert torch.equal(dyf, want)

    q, scale = _abi.quantize_f8(x)
    qf = torch.empty(2 * apart + cols, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).as_strided((3, cols), (apart, 1))
    sf = torch.empty_like(scale)
    _abi.check(lib.tvk_quantize_f8(C.byref(_abi.make_quantize_f8_desc(far(x, 0), qf, sf, 1, stream))))
    assert torch.equal(qf.contiguous().view(torch.uint8), q.view(torch.uint8)) and torch.equal(sf, scale)
    w, w_scale = _abi.quantize_f8(torch.randn((cols, cols), generator=gen).bfloat16().cuda(), 128)
    want = _abi.gemm_f8(x, None, w, w_scale)
    out = far(torch.zeros_like(x), 1)
    for a, s in ((far(x, 0), None), (qf, scale)):   # (as the rows, and as their 8 bits)
        out.zero_()
        _abi.check(lib.tvk_gemm_f8(C.byref(_abi.make_gemm_f8_desc(a, s, w, w_scale, out, stream=stream))))
        assert torch.equal(out, want)
    tall = torch.randn((70, 256), generator=gen).bfloat16().cuda()   # the tiled kernel's output
    wide = memory[0].as_strided((70, 256), (30_000_000, 1))
    few, few_scale = _abi.quantize_f8(torch.randn((256, 256), generator=gen).bfloat16().cuda(), 128)
    _abi.check(lib.tvk_gemm_f8(C.byref(_abi.make_gemm_f8_desc(tall, None, few, few_scale, wide, stream=stream))))
    assert torch.equal(wide, _abi.gemm_f8(tall, None, few, few_scale))
