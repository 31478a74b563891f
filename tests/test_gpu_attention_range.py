"""Attention over 8-bit caches where the weights' reference and that of weights times scales lie far apart: scores that jump, values that are
all zeros, scales of very different size. Bounds are derived in attention_helpers; the caches hold one number of each key, so that scores
are what a test says."""
import math

import pytest

pytestmark = pytest.mark.gpu

LN2 = math.log(2.0)
GAINS = [1.0, 0.75, -1.0, 0.1]  # of the query heads: each sees the scores times its own


def _cache(fmt, dim, scores, values, page=16):
    """One sequence of len(scores) tokens, one key head: key j is scores[j] in its first place, value j is values[j]."""
    import torch

    from attention_helpers import POOLS, Cache, quantise64

    n = len(scores)
    cache = Cache(fmt, 1, dim, page, 1, -(-n // page))
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    pages, slots = cache.place(torch.zeros_like(at), at)
    keys = torch.zeros(n, 1, dim, device="cuda")
    keys[:, 0, 0] = scores
    raw = torch.int16 if fmt == "bf16" else torch.uint8
    for side, x in ((0, keys), (1, values)):
        codes, scales = quantise64(x, fmt)
        cache.pools[side].view(raw)[pages, :, slots] = codes.to(POOLS[fmt]).view(raw)
        if scales is not None:
            cache.scales[side][pages, :, slots] = scales
    return cache


def _queries(dim, q_tokens):
    import torch

    q = torch.zeros(q_tokens, len(GAINS), dim, device="cuda")
    q[:, :, 0] = torch.tensor(GAINS, device="cuda")
    return q


def _attend(rt, cache, n, q, scale=1.0):
    import torch

    from attention_helpers import kind

    out = torch.full(q.shape, math.nan, device="cuda")
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    width = q.shape[1] * q.shape[2]
    torch.cuda.synchronize()
    rt.attention_device(cache.c, cache.t, lengths.data_ptr(), q.data_ptr(), kind("f32"), width, q.shape[1], q.shape[0], scale, out.data_ptr(), kind("f32"), width)
    rt.device_status()
    return out


def _check(rt, cache, n, q):
    """Two things are added to the bound: weights below 2^-126 of the row's largest one count as nothing, which takes that much of all values from
    the result at most; and weights times scales, multiplied by 2^126 at most, are whole numbers (int8) off by half, or e4m3 halves off by 2^-25."""
    import torch

    from attention_helpers import POOLS, attention64, rounded

    out = _attend(rt, cache, n, q)
    ref, bound = attention64(cache, [n], q, q.shape[0], 1.0)
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    values, raw, _ = cache.held(1, torch.zeros_like(at), at)
    nothing = 2.0 ** -126 * values.abs().sum(0)
    steps = 2.0 ** (-127 if cache.fmt == "int8" else -151) * raw.view(POOLS[cache.fmt]).double().abs().sum(0)
    off, most = (out.double() - ref).abs(), rounded(bound + nothing + steps, ref, "f32") - 1e-37 + 1e-43
    assert bool((off <= most).all()), (float((off / most).max()), out.isnan().sum().item())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,q_tokens", [(64, 1), (128, 3), (256, 1)])
def test_small_values(runtime, fmt, dim, q_tokens):
    """Scales far below those of ordinary values: of all tokens, and of those seen beside a token that takes nearly all and has values of zeros."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(dim + q_tokens)
    q = _queries(dim, q_tokens)
    for n in (40, 300, 9000):
        scores, values = torch.rand(n, generator=gen, device="cuda"), torch.randn(n, 1, dim, generator=gen, device="cuda")
        for size in (-60, -84, -94, -100, -106):
            _check(runtime, _cache(fmt, dim, scores, values * 2.0 ** size), n, q)
        values[33] = 0.0
        for jump in (60, 90, 100, 110, 118):
            scores[33] = jump * LN2
            _check(runtime, _cache(fmt, dim, scores, values), n, q)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 256])
def test_a_large_value_that_hardly_counts_among_small_ones(runtime, fmt, dim):
    """Scales of 2^-100 with weights of one, and one of 2^90 with a weight of 2^-60 to 2^-125."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(dim)
    q = _queries(dim, 1)
    for n, large in ((300, 7), (300, 290), (9000, 8999)):
        values = torch.randn(n, 1, dim, generator=gen, device="cuda")
        values = values * torch.where(torch.arange(n, device="cuda")[:, None, None] == large, 2.0 ** 95, 2.0 ** -95)
        scores = torch.rand(n, generator=gen, device="cuda")
        for fall in (60, 90, 110, 125):
            scores[large] = -fall * LN2
            _check(runtime, _cache(fmt, dim, scores, values), n, q)
