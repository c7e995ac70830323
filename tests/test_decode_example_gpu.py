"""examples/decode.py: the captured step gives the eager steps' tokens, bit for bit where both are given the same bound."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

import torchvulkan_amd  # noqa: F401  (registers the vulkan device)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("length,count", [(37, 12), (700, 20)])
def test_captured_tokens_are_the_eager_ones(gpu, cache_dtype, length, count):
    spec = importlib.util.spec_from_file_location("decode_example", Path(__file__).resolve().parent.parent / "examples" / "decode.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    model = example.Decoder(layers=2, dim=256, heads=4, heads_kv=2, hidden=512, vocab=500)
    prompts = torch.randint(0, 500, (3, length), generator=torch.Generator().manual_seed(0)).cuda()
    captured = example.generate(model, prompts, count, cache_dtype, capture=True)[0]
    cache = model.cache(3, length + count, dtype=cache_dtype)
    cache.extend(length)
    token = model(prompts, cache).argmax(-1, keepdim=True)
    eager = [token]
    for _ in range(count - 1):
        cache.extend(1)
        token = model(token, cache, max_len=length + count).argmax(-1, keepdim=True)
        eager.append(token)
    assert torch.equal(captured, torch.cat(eager, 1))
