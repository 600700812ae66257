"""Writes into 8-bit caches of many key heads, up to 1024 rows and more: each head's bytes and range as in a cache of that head alone (GPU)."""

import pytest
import torch

import qr_v2_b200_kernel_b200 as qr

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, dim", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("heads", [9, 12, 32])
@pytest.mark.parametrize("rows", [1, 3, 7, 8, 9, 40, 300, 1024, 1500])
def test_many_heads(rows, heads, dim, dtype):
    # single tokens of many pages and runs of one, into pages that hold some already
    page, pages = 64, 40
    g = torch.Generator(device="cuda").manual_seed(rows + heads)
    whole = qr.kv8_cache(pages, page, heads, dim, dtype=dtype)
    alone = [qr.kv8_cache(pages, page, 1, dim, dtype=dtype) for _ in range(heads)]
    every = torch.arange(pages * page, device="cuda")
    some = torch.randperm(pages * page, generator=g, device="cuda")[:rows]
    run = (torch.arange(rows, device="cuda") + 70) % (pages * page)
    for turn, slots in enumerate((every, some, run)):
        k, v = (((1 + turn) * torch.randn(len(slots), heads, dim, generator=g, device="cuda")).to(dtype) for _ in range(2))
        qr.kv8_write(whole, k, v, slots)
        for h, cache in enumerate(alone):
            qr.kv8_write(cache, k[:, h : h + 1], v[:, h : h + 1], slots)
    assert torch.equal(whole.range, torch.cat([c.range for c in alone], 1))
    assert torch.equal(whole.data, torch.cat([c.data for c in alone], 1))
