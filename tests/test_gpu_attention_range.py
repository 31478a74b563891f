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
    """Two things are added to the bound. Weights are relative to a whole power of two, which lies up to one power above the row's largest score:
    those below 2^-126 count as nothing, which takes 2^-125 of all values from the result at most. Weights times scales, multiplied by 2^126 at
    most, are whole numbers (int8) off by half, 2^-127, or e4m3 halves off by 2^-25, 2^-151: twice that of the largest weight."""
    import torch

    from attention_helpers import POOLS, attention64, rounded

    out = _attend(rt, cache, n, q)
    ref, bound = attention64(cache, [n], q, q.shape[0], 1.0)
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    values, raw, _ = cache.held(1, torch.zeros_like(at), at)
    nothing = 2.0 ** -125 * values.abs().sum(0)
    steps = 2.0 ** (-126 if cache.fmt == "int8" else -150) * raw.view(POOLS[cache.fmt]).double().abs().sum(0)
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


# one block's second step of 256 tokens with one token and with many; items that several blocks work on, in one step and in two
PLACES = [(257, 256), (300, 270), (9000, 8999), (60011, 330), (60011, 60010)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,q_tokens", [(64, 1), (64, 4), (128, 6), (256, 1), (256, 4)])
@pytest.mark.parametrize("zero", [True, False])
def test_a_score_that_jumps(runtime, fmt, dim, q_tokens, zero):
    """A token far above those before it, in powers of two; its value is all zeros or like the others."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(dim + q_tokens)
    q = _queries(dim, q_tokens)
    for n, peak in PLACES:
        scores = torch.rand(n, generator=gen, device="cuda")
        values = torch.randn(n, 1, dim, generator=gen, device="cuda")
        if zero:
            values[peak] = 0.0
        for jump in (30, 60, 97, 100, 120, 128, 160, 200, 1000):
            scores[peak] = jump * LN2
            _check(runtime, _cache(fmt, dim, scores, values), n, q)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 256])
def test_nothing_but_zeros_at_the_top(runtime, fmt, dim):
    """Scores that rise from step to step with values of zeros, then ordinary values again, and only zeros."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(dim)
    n = 520  # three steps of one block
    scores = torch.rand(n, generator=gen, device="cuda") + (torch.arange(n, device="cuda") // 100) * 40 * LN2
    q = _queries(dim, 2)
    for first, last in ((256, 512), (256, n), (0, 256), (0, n)):
        values = torch.randn(n, 1, dim, generator=gen, device="cuda")
        values[first:last] = 0.0
        _check(runtime, _cache(fmt, dim, scores, values), n, q)


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "bf16"])
@pytest.mark.parametrize("dim", [64, 256])
def test_scores_that_24_bits_hold_in_steps_above_one(runtime, fmt, dim):
    """The peak takes all where it is seen from above, and nothing (the others are equal) where its score is negative."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(dim)
    q = _queries(dim, 1)
    for n, peak in PLACES + [(300, 3), (9000, 5)]:
        values = torch.randn(n, 1, dim, generator=gen, device="cuda")
        for size in (2.0 ** 24, 2.0 ** 27, 2.0 ** 31, 2.0 ** 40, 2.0 ** 100):
            scores = torch.zeros(n, device="cuda")
            scores[peak] = size
            cache = _cache(fmt, dim, scores, values)
            out = _attend(runtime, cache, n, q)
            at = torch.arange(n, dtype=torch.int32, device="cuda")
            held = cache.held(1, torch.zeros_like(at), at)[0][:, 0]
            # a weight of its own: two roundings of it, three of the sum of digits, or two of halves, and those of the quotient
            off = (out[0, [0, 1, 3]].double() - held[peak]).abs()
            assert bool((off <= 2.0 ** -16 * held[peak].abs()).all()), (n, peak, size)
            others = torch.cat([held[:peak], held[peak + 1:]])
            off = (out[0, 2].double() - others.mean(0)).abs()
            assert bool((off <= 2.0 ** -15 * others.abs().mean(0)).all()), (n, peak, size)


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "bf16"])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("size", [-90, -40, 60, 100])
def test_queries_far_from_one(runtime, fmt, dim, size):
    """Queries of 2^size times the usual and keys of as much less: the scores are what they always are."""
    import torch

    from attention_helpers import Cache

    n, q_tokens, heads = 400, 3, 6
    cache = Cache(fmt, 1, dim, 16, 1, n // 16)
    cache.fill([n], dim, k_gain=2.0 ** -size)
    gen = torch.Generator(device="cuda").manual_seed(dim)
    q = torch.randn(q_tokens, heads, dim, generator=gen, device="cuda") * 2.0 ** size * dim ** -0.5
    _check(runtime, cache, n, q)


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "bf16"])
@pytest.mark.parametrize("dim,heads", [(64, 1), (64, 16), (128, 1), (128, 16), (256, 1), (256, 16), (256, 24)])
def test_sums_over_many_tokens_of_one_block(runtime, fmt, dim, heads):
    """More long sequences than blocks, all reading the same pages. Queries of zero: weights of exactly one, so that the result is the mean of positive
    values, and off by what its sum loses: steps of 256 tokens at most, in which 16 additions of 16 tokens or less lose a last place of 24
    bits each, 2^-23; the sum of steps, n / 128 additions that are rounded, 2^-24 each; 2^-21 for joining, the quotient and a weight's halves."""
    import torch

    from attention_helpers import POOLS, Cache

    n, sequences = 30000, 160
    cache = Cache(fmt, 1, dim, 16, sequences, n // 16, share=True)
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    pages, slots = cache.place(torch.zeros_like(at), at)
    gen = torch.Generator(device="cuda").manual_seed(dim)
    # of very different size, so that their sum does not fit 24 bits
    values = (8 + torch.randint(0, 8, (n, 1, dim), generator=gen, device="cuda")) * torch.exp2(-torch.randint(0, 9, (n, 1, dim), generator=gen, device="cuda").float())
    for side, x in ((0, torch.ones_like(values)), (1, values)):
        codes = (x.ceil() if fmt == "int8" else x).to(POOLS[fmt])
        cache.pools[side].view(torch.int16 if fmt == "bf16" else torch.uint8)[pages, :, slots] = codes.view(torch.int16 if fmt == "bf16" else torch.uint8)
        if cache.scales:
            cache.scales[side][pages, :, slots] = 0.3
    want = cache.held(1, torch.zeros_like(at), at)[0].mean(0)[0]
    from attention_helpers import kind

    q = torch.zeros(sequences, heads, dim, device="cuda")
    out = torch.full_like(q, math.nan)
    lengths = torch.full((sequences,), n, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    runtime.attention_device(cache.c, cache.t, lengths.data_ptr(), q.data_ptr(), kind("f32"), heads * dim, heads, 1, 1.0, out.data_ptr(), kind("f32"), heads * dim)
    runtime.device_status()
    off = ((out.double() - want) / want).abs().max().item()
    assert off <= 16 * 2.0 ** -23 + n / 128 * 2.0 ** -24 + 2.0 ** -21, off
