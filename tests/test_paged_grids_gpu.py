"""Calls of more workgroups than one dimension of a grid holds (2^32 threads): tvk_paged_append and tvk_paged_attention take
them as they take smaller ones."""
from __future__ import annotations

import pytest
import torch

from torchvulkan_amd import _abi

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


# sequences of one key each: their values are the result. Rows of the general kernel; segments past what the MFMA kernel's
# launches hold, of a workgroup and of a wave, which the general kernel takes.
@pytest.mark.parametrize("batch,heads,dim,max_len", [((1 << 18) + 1, 64, 8, 1), ((1 << 18) + 1, 64, 16, 200), ((1 << 20) + 1, 64, 16, 1)])
def test_attention_of_many_rows(gpu, batch, heads, dim, max_len):
    g = torch.Generator(device=DEV).manual_seed(0)
    k, v = (torch.randn((5, 1, heads, dim), generator=g, device=DEV).to(torch.float16) for _ in range(2))
    table = (torch.arange(batch, device=DEV) % 5).to(torch.int32)[:, None].expand(batch, 1).contiguous()
    q = torch.randn((batch, 1, 1, dim), generator=g, device=DEV).to(torch.float16).expand(batch, 1, heads, dim)
    table = torch.cat([table, torch.full((batch, 199), -1, dtype=torch.int32, device=DEV)], 1) if max_len > 1 else table
    out, lse = _abi.paged_attention(q, k, v, torch.ones(batch, dtype=torch.int32, device=DEV), table, max_len=max_len)
    for i in range(5):
        assert torch.equal(out[i::5], v[i][None].expand(out[i::5].shape))
    assert lse.isfinite().all()


def test_append_of_many_tokens(gpu):
    tokens, page, dim = (1 << 26) + 3, 4096, 8
    pages = -(-tokens // page)
    k, v = (torch.randn((1, tokens, 1, dim), dtype=torch.float16, device=DEV) for _ in range(2))
    kc, vc = (torch.zeros((pages, page, 1, dim), dtype=torch.float16, device=DEV) for _ in range(2))
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    _abi.paged_append(None, k, v, kc, vc, torch.tensor([tokens], dtype=torch.int32, device=DEV), table)
    for cache, x in ((kc, k), (vc, v)):
        flat = cache.view(-1, dim)
        assert torch.equal(flat[:tokens], x[0, :, 0]) and flat[tokens:].eq(0).all()
