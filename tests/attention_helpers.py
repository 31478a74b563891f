"""Plain forms in 64 bits, and the caches that the tests of the attention operators build."""
from __future__ import annotations

import math
from fractions import Fraction

import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
POOLS = {"bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}


def kind(name):
    from qwen38_metal_b200 import capi

    return {"f32": capi.Q4B_F32, "bf16": capi.Q4B_BF16}[name]


class Cache:
    """Pools, scales, page table and their descriptions. `order`: how tokens, heads and pages lie in memory, with `gap` bytes
    between rows, heads and pages. Everything in the pools starts as `fill` (a byte), scales as NaN: nothing may depend on it."""

    def __init__(self, fmt, kv_heads, dim, page, sequences, per, spare=2, order="phtd", gap=0, fill=0xff, seed=0, share=False):
        from qwen38_metal_b200 import KvCache, KvTable

        self.fmt, self.kv_heads, self.dim, self.page, self.sequences, self.per = fmt, kv_heads, dim, page, sequences, per
        self.pages = (per if share else sequences * per) + spare
        size = 2 if fmt == "bf16" else 1
        count = {"p": self.pages, "h": kv_heads, "t": page}
        stride, extent = {}, dim * size + gap
        for axis in reversed(order[:3]):
            stride[axis] = extent
            extent = extent * count[axis] + gap
        self.stride = stride
        self.raw = [torch.full((extent,), fill, dtype=torch.uint8, device="cuda") for _ in range(2)]
        self.pools = [torch.as_strided(r.view(POOLS[fmt]), (self.pages, kv_heads, page, dim),
                                       (stride["p"] // size, stride["h"] // size, stride["t"] // size, 1)) for r in self.raw]
        self.scales = None
        if fmt != "bf16":
            self.scales = [torch.full((self.pages, kv_heads, page), math.nan, device="cuda") for _ in range(2)]
        gen = torch.Generator().manual_seed(seed + 77)
        numbers = torch.randperm(self.pages, generator=gen)
        self.table = (numbers[:per].repeat(sequences, 1) if share else numbers[:sequences * per].view(sequences, per)).to(torch.int32).cuda()
        self.c = KvCache(fmt, kv_heads, dim, page, self.pages, self.raw[0].data_ptr(), self.raw[1].data_ptr(),
                         self.scales[0].data_ptr() if self.scales else 0, self.scales[1].data_ptr() if self.scales else 0,
                         stride["p"], stride["h"], stride["t"])
        self.t = KvTable(self.table.data_ptr(), sequences, per)

    def place(self, sequences, positions):
        return self.table[sequences.long(), positions.long() // self.page].long(), positions.long() % self.page

    def held(self, side, sequences, positions):
        """What the cache holds for these tokens, [tokens][kv heads][dim] in 64 bits, and codes and scales."""
        page, slot = self.place(sequences, positions)
        raw = self.pools[side].view(torch.int16 if self.fmt == "bf16" else torch.uint8)[page, :, slot]
        codes = raw.view(POOLS[self.fmt]).double()
        if self.fmt == "bf16":
            return codes, raw, None
        scales = self.scales[side][page, :, slot]
        return codes * scales.double()[..., None], raw, scales

    def fill(self, lengths, seed, k_gain=1.0, vary=0.5):
        """Random keys and values for the first lengths[s] tokens of every sequence, put there by torch."""
        gen = torch.Generator(device="cuda").manual_seed(seed)
        sequences = torch.cat([torch.full((n,), s, dtype=torch.int32) for s, n in enumerate(lengths)]).cuda()
        positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in lengths]).cuda()
        if sequences.numel() == 0:
            return
        page, slot = self.place(sequences, positions)
        for side, gain in ((0, k_gain), (1, 1.0)):
            x = gain * torch.randn(len(sequences), self.kv_heads, self.dim, generator=gen, device="cuda")
            x = x * torch.exp(vary * torch.randn(len(sequences), self.kv_heads, 1, generator=gen, device="cuda"))
            codes, scales = quantise64(x, self.fmt)
            self.pools[side].view(torch.int16 if self.fmt == "bf16" else torch.uint8)[page, :, slot] = \
                codes.to(POOLS[self.fmt]).view(torch.int16 if self.fmt == "bf16" else torch.uint8)
            if scales is not None:
                self.scales[side][page, :, slot] = scales


def quantise64(x, fmt):
    """Codes (as numbers) and fp32 scales by the definition: the code nearest to x / scale, ties to even, quotients in 64 bits."""
    x = x.float()
    if fmt == "bf16":
        return x.to(torch.bfloat16), None
    amax = x.abs().amax(-1)
    scale = (amax.double() / TOP[fmt]).float()  # rounding a 53-bit quotient of two 24-bit numbers again is harmless
    finite = torch.isfinite(amax)
    ratio = torch.where((scale > 0)[..., None] & finite[..., None], x.double() / scale.double()[..., None], 0.0)
    scale = torch.where(finite, scale, math.nan)
    if fmt == "int8":
        return ratio.round().clamp(-127, 127), scale
    step = torch.ldexp(torch.ones_like(ratio), torch.frexp(ratio.abs().clamp(min=2.0 ** -6))[1] - 4)
    return ((ratio / step).round() * step).clamp(-448, 448), scale


def exact_angles(positions, freq):
    """positions x freq modulo a turn, from whole numbers: 64 bits are too few for an angle of 2^31 rad."""
    turn = 2 * Fraction(31415926535897932384626433832795028841971693993751, 10 ** 49)
    return torch.tensor([[float(Fraction(float(f)) * p % turn) for f in freq] for p in positions.tolist()], dtype=torch.float64).cuda()


def turned64(x, positions, freq, factor, layout, exact=False):
    """x [tokens][heads][dim] turned, in 64 bits; and for every value the size |a| + |b| of its pair (0 where it is not turned)."""
    z = x.double().clone()
    size = torch.zeros_like(z)
    pairs = len(freq)
    i = torch.arange(pairs, device=x.device)
    first, second = (i, i + pairs) if layout == "half" else (2 * i, 2 * i + 1)
    angle = exact_angles(positions, freq) if exact else positions.double()[:, None] * torch.as_tensor(freq, device=x.device, dtype=torch.float64)
    c, s = factor * torch.cos(angle)[:, None], factor * torch.sin(angle)[:, None]
    a, b = z[..., first].clone(), z[..., second].clone()
    z[..., first], z[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(factor)
    return z, size


def attention64(cache, lengths, q, q_tokens, scale):
    """Attention in 64 bits and a bound for the error of one that keeps the two factors of each product to 16 bits.

    |q - q'| <= 2^-16 |q| (two bf16 numbers: each rounding is off by at most 2^-8 of what it rounds), and sums of up to 256
    products in 32 bits add less than 256 * 2^-24 = 2^-16 of the sum of magnitudes, scaling and exponential 2^-16 of the score
    at most; so a score is off by d = 2^-14 scale sum |q k| at most, its weight by e^d - 1 < 1.06 d (d < 0.1) and the mean of the
    values by twice that of the mean of their magnitudes. Weights kept to 16 bits: 2^-16 of it; 32-bit sums of n terms in
    blocks of 16 tokens, then of blocks: 2^-24 (16 + n / 16), and of partial results less than 2^-17.

    8-bit caches keep halves in fp16, whose smallest step is 2^-24: queries are scaled to a largest value of 1 or more, so a query is
    off by 2^-16 of itself or by 2^-25 of the largest one, whichever is more: that adds 2^-25 scale max|q| sum |k| to d. Weights times
    scales w_j = p_j scale_j are, for int8, whole numbers of which the largest one so far is 2^25 or more: off by half at most, 2^-26 of
    the largest one; for e4m3 scaled so that the largest one is 2^10 or more, and off by 2^-16 of themselves or by 2^-25 2^-10 of it.
    That adds 2^-26, 2^-35 max w sum |code| to the result."""
    rows, heads, dim = q.shape
    group = heads // cache.kv_heads
    out = torch.zeros(rows, heads, dim, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    for s, n in enumerate(lengths):
        if n <= 0:
            continue
        at = torch.arange(n, dtype=torch.int32, device="cuda")
        seq = torch.full_like(at, s)
        k = cache.held(0, seq, at)[0]
        v, raw, v_scales = cache.held(1, seq, at)
        for i in range(q_tokens):
            seen = n - q_tokens + 1 + i
            if seen <= 0:
                continue
            x = q[s * q_tokens + i].double().view(cache.kv_heads, group, dim)
            score = torch.einsum("hgd,thd->hgt", x, k[:seen]) * scale
            size = torch.einsum("hgd,thd->hgt", x.abs(), k[:seen].abs()) * abs(scale)
            p = torch.softmax(score, -1)
            steps = 0.0
            if v_scales is not None:
                size = size + 2.0 ** -11 * abs(scale) * torch.einsum("hg,th->hgt", x.abs().amax(-1), k[:seen].abs().sum(-1))
                codes = raw[:seen].view(POOLS[cache.fmt]).double().abs().sum(0)
                steps = 2.0 ** (-26 if cache.fmt == "int8" else -35) * (p * v_scales[:seen].double().T[:, None]).amax(-1)[..., None] * codes[:, None]
                steps = steps.reshape(heads, dim)
            out[s * q_tokens + i] = torch.einsum("hgt,thd->hgd", p, v[:seen]).reshape(heads, dim)
            mean = torch.einsum("hgt,thd->hgd", p, v[:seen].abs()).reshape(heads, dim)
            off = 2.12 * 2.0 ** -14 * size.amax(-1) + 2.0 ** -16 + 2.0 ** -24 * (16 + seen / 16) + 2.0 ** -17
            assert float((2.0 ** -14 * size.amax(-1)).max()) < 0.1
            bound[s * q_tokens + i] = mean * off.reshape(heads, 1) + steps
    return out, bound


def rounded(bound, ref, out):
    """The bound with the rounding to the output's type: half a step of bf16 is 2^-8 of the value."""
    return bound + (ref.abs() + bound) * (2.0 ** -8 if out == "bf16" else 2.0 ** -24) + 1e-37


def strided(shape, stride, dtype, fill):
    """A [tokens][width] view whose rows are `stride` values apart in memory filled with `fill`."""
    tokens, width = shape
    base = torch.full((tokens * stride,), fill, dtype=dtype, device="cuda")
    return base, base.view(tokens, stride)[:, :width]
