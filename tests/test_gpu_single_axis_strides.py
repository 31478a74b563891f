"""Caches of one key head, one page or one head and page: the stride along an axis of one is nothing that a call looks at."""
import math
from dataclasses import replace

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "bf16"])
@pytest.mark.parametrize("dim", [48, 64, 256])
@pytest.mark.parametrize("kv_heads,pages", [(1, 5), (3, 1), (1, 1)])
def test_strides_of_axes_of_one(runtime, fmt, dim, kv_heads, pages):
    import torch

    from attention_helpers import Cache, kind

    page, n = 32, 32 * min(pages, 4) - 3
    cache = Cache(fmt, kv_heads, dim, page, 1, min(pages, 4), spare=pages - min(pages, 4))
    cache.fill([n], 3)
    gen = torch.Generator(device="cuda").manual_seed(dim)
    heads = 2 * kv_heads
    q = torch.randn(1, heads, dim, generator=gen, device="cuda")
    k, v = (torch.randn(n, kv_heads, dim, generator=gen, device="cuda") for _ in range(2))
    lengths, positions = torch.tensor([n], dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    f32, width = kind("f32"), heads * dim

    def attend(c):
        out = torch.full_like(q, math.nan)
        runtime.attention_device(c, cache.t, lengths.data_ptr(), q.data_ptr(), f32, width, heads, 1, 0.1, out.data_ptr(), f32, width)
        runtime.device_status()
        return out

    def written(c):
        back = [torch.full_like(k, math.nan) for _ in range(2)]
        runtime.kv_write_device(c, cache.t, positions.data_ptr(), 0, n, k.data_ptr(), kv_heads * dim, v.data_ptr(), kv_heads * dim, f32)
        runtime.kv_read_device(c, cache.t, positions.data_ptr(), 0, n, back[0].data_ptr(), kv_heads * dim, back[1].data_ptr(), kv_heads * dim, f32)
        runtime.device_status()
        return back

    given = (cache.stride["t"], cache.stride["h"], cache.stride["p"])
    held, want = None, attend(cache.c)
    for other in (0, 16, 1 << 39):
        strides = (given[0], other if kv_heads == 1 else given[1], other if pages == 1 else given[2])
        c = replace(cache.c, token_stride=strides[0], head_stride=strides[1], page_stride=strides[2])
        assert torch.equal(attend(c), want), strides
    held = written(cache.c)
    want = attend(cache.c)
    for other in (0, 16, 1 << 39):
        strides = (given[0], other if kv_heads == 1 else given[1], other if pages == 1 else given[2])
        c = replace(cache.c, token_stride=strides[0], head_stride=strides[1], page_stride=strides[2])
        assert all(torch.equal(a, b) for a, b in zip(written(c), held)) and torch.equal(attend(c), want), strides
