"""Attention of new tokens over the paged cache against the formula in 64 bits; bounds are derived in attention_helpers."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _attend(rt, cache, lengths, q, q_tokens, scale, out, names, heads, q_stride=None, out_stride=None, stream=0):
    from attention_helpers import kind

    width = heads * cache.dim
    rt.attention_device(cache.c, cache.t, lengths.data_ptr(), q.data_ptr(), kind(names[0]), q_stride or width, heads, q_tokens, scale, out.data_ptr(), kind(names[1]),
                        out_stride or width, stream)


def _case(rt, fmt, lengths, q_tokens, heads, kv_heads, dim, page, names, seed=1, q_gain=1.0, per=None, check=True, **more):
    import torch

    from attention_helpers import DTYPES, Cache, attention64, rounded

    per = per or max(1, max((n + page - 1) // page for n in lengths))
    cache = Cache(fmt, kv_heads, dim, page, len(lengths), per, seed=seed, **more)
    cache.fill(lengths, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = (q_gain * torch.randn(len(lengths) * q_tokens, heads, dim, generator=gen, device="cuda")).to(DTYPES[names[0]])
    out = torch.full(q.shape, math.nan, dtype=DTYPES[names[1]], device="cuda")
    device_lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    scale = dim ** -0.5
    _attend(rt, cache, device_lengths, q, q_tokens, scale, out, names, heads)
    rt.device_status()
    if check:
        ref, bound = attention64(cache, lengths, q, q_tokens, scale)
        off = (out.double() - ref).abs()
        assert bool((off <= rounded(bound, ref, names[1])).all()), float((off / rounded(bound, ref, names[1])).max())
    return cache, device_lengths, q, out, scale


# lengths around tiles and pages, none at all, one
RAGGED = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200, 511, 1025]


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(24, 4, 256, 16), (8, 1, 128, 48), (3, 3, 64, 32), (5, 1, 16, 16), (14, 2, 80, 64), (16, 1, 192, 16), (40, 2, 96, 256), (8, 8, 256, 16)])
@pytest.mark.parametrize("names", [("f32", "f32"), ("bf16", "bf16")])
def test_ragged_batch(runtime, fmt, heads, kv_heads, dim, page, names):
    _case(runtime, fmt, RAGGED, 1, heads, kv_heads, dim, page, names)


@pytest.mark.parametrize("fmt", ["int8", "bf16"])
@pytest.mark.parametrize("q_tokens,heads,kv_heads,dim", [(2, 24, 4, 256), (4, 24, 4, 256), (7, 6, 2, 64), (16, 4, 4, 128), (16, 24, 2, 32), (3, 8, 8, 112)])
def test_draft_tokens(runtime, fmt, q_tokens, heads, kv_heads, dim):
    """Every token sees itself and what stands before it; a sequence shorter than its new tokens leaves the first rows empty."""
    lengths = [q_tokens, 1, 0, q_tokens + 1, 16 + q_tokens // 2, 64, 65 + q_tokens, 300]
    _, _, _, out, _ = _case(runtime, fmt, lengths, q_tokens, heads, kv_heads, dim, 16, ("f32", "f32"))
    rows = out.view(len(lengths), q_tokens, heads, dim)
    assert bool((rows[1, :q_tokens - 1] == 0).all()) and bool((rows[2] == 0).all()) and bool((rows[1, -1] != 0).any())


@pytest.mark.parametrize("fmt,lengths,heads,kv_heads,dim,page", [("int8", [50001], 24, 4, 256, 16), ("bf16", [30011], 12, 2, 128, 64), ("e4m3", [40000, 3], 8, 1, 64, 48),
                                                                ("int8", [20000, 1, 0, 7777], 24, 4, 256, 256)])
def test_long_contexts_are_split_and_joined(runtime, fmt, lengths, heads, kv_heads, dim, page):
    _case(runtime, fmt, lengths, 1, heads, kv_heads, dim, page, ("f32", "f32"), q_gain=2.0)


# 9 to 48 query rows of a key head, which are multiplied 16 or 24 at a time, the last of them partly empty
WIDE = [("bf16", 2, 24, 4, 256), ("bf16", 4, 24, 4, 256), ("bf16", 5, 8, 1, 256), ("bf16", 3, 8, 2, 128), ("bf16", 16, 3, 1, 48), ("e4m3", 4, 8, 2, 128), ("e4m3", 3, 5, 1, 64),
        ("int8", 9, 2, 1, 64), ("int8", 2, 24, 3, 128), ("int8", 3, 24, 4, 256), ("e4m3", 3, 24, 4, 256)]


@pytest.mark.parametrize("fmt,q_tokens,heads,kv_heads,dim", WIDE)
def test_more_rows_of_a_key_head(runtime, fmt, q_tokens, heads, kv_heads, dim):
    _case(runtime, fmt, RAGGED, q_tokens, heads, kv_heads, dim, 16, ("f32", "f32"))
    _case(runtime, fmt, [20011, 7, 1031], q_tokens, heads, kv_heads, dim, 64, ("bf16", "bf16"), q_gain=2.0)


@pytest.mark.parametrize("fmt,q_tokens,heads,kv_heads,dim", WIDE)
def test_numbers_that_are_not_finite_among_more_rows(runtime, fmt, q_tokens, heads, kv_heads, dim):
    import torch

    group, n = heads // kv_heads, 40
    for where in ("k", "v", "q"):
        cache, lengths, q, out, scale = _case(runtime, fmt, [n, n], q_tokens, heads, kv_heads, dim, 16, ("f32", "f32"))
        page, slot = cache.place(torch.tensor([0], device="cuda"), torch.tensor([n - 2], device="cuda"))
        good, last = out.clone(), kv_heads - 1
        if where == "q":
            q[1, heads - 1, 5] = math.nan
        elif fmt == "bf16":
            cache.pools["kv".index(where)][page, last, slot, 3] = math.nan
        else:
            cache.scales["kv".index(where)][page, last, slot] = math.nan
        _attend(runtime, cache, lengths, q, q_tokens, scale, out, ("f32", "f32"), heads)
        runtime.device_status()
        bad = torch.zeros_like(out, dtype=torch.bool)
        if where == "q":
            bad[1, heads - 1] = True
        else:
            # the last two tokens of sequence 0 see position n - 2
            bad[max(q_tokens - 2, 0):q_tokens, last * group:(last + 1) * group, slice(3, 4) if where == "v" and fmt == "bf16" else slice(None)] = True
        assert torch.equal(torch.isnan(out), bad)
        assert torch.equal(out[~bad], good[~bad])


@pytest.mark.parametrize("names", [("f32", "bf16"), ("bf16", "f32")])
def test_many_sequences(runtime, names):
    lengths = [(i * 37) % 150 for i in range(700)]
    _case(runtime, "int8", lengths, 1, 6, 2, 64, 16, names)


@pytest.mark.parametrize("fmt", ["int8", "bf16"])
def test_more_sequences_than_a_block_has_threads(runtime, fmt):
    _case(runtime, fmt, [0] * 3000 + [40] + [0] * 2000 + [17, 0, 3], 2, 4, 2, 32, 16, ("f32", "f32"))


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "bf16"])
def test_what_lies_behind_a_sequence_is_not_looked_at(runtime, fmt):
    """Unused places of the pools and their scales hold NaNs and infinities (they do everywhere in these tests); so do unused
    entries of the page table, which name no page."""
    import torch

    from attention_helpers import attention64, rounded

    cache, lengths, q, out, scale = _case(runtime, fmt, [1, 19, 0, 50], 1, 6, 2, 64, 16, ("f32", "f32"), per=9)
    used = torch.tensor([1, 2, 0, 4], device="cuda")
    cache.table[torch.arange(9, device="cuda")[None] >= used[:, None]] = 1 << 29
    first = out.clone()
    for byte in (0x7f, 0x80, 0x00):
        # rows without a token take any value: 0x7f7f and 0x7f80 bf16 are a large number and infinity, 0x7f e4m3 a NaN
        fresh = [r.clone() for r in cache.raw]
        sequences = torch.cat([torch.full((n,), s, dtype=torch.int32) for s, n in enumerate([1, 19, 0, 50])]).cuda()
        positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in [1, 19, 0, 50]]).cuda()
        page, slot = cache.place(sequences, positions)
        for side in range(2):
            raw = cache.pools[side].view(torch.int16 if fmt == "bf16" else torch.uint8)
            kept = raw[page, :, slot].clone()
            cache.raw[side].fill_(byte)
            raw[page, :, slot] = kept
            if cache.scales:
                kept = cache.scales[side][page, :, slot].clone()
                cache.scales[side].fill_({0x7f: math.inf, 0x80: -math.inf, 0: 0.0}[byte])
                cache.scales[side][page, :, slot] = kept
        _attend(runtime, cache, lengths, q, 1, scale, out, ("f32", "f32"), 6)
        runtime.device_status()
        assert torch.equal(out, first)
        for side in range(2):
            cache.raw[side].copy_(fresh[side])


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "bf16"])
def test_numbers_that_are_not_finite_stay_in_their_rows(runtime, fmt):
    import torch

    for where in ("k", "v", "q"):
        cache, lengths, q, out, scale = _case(runtime, fmt, [40, 40], 2, 6, 2, 64, 16, ("f32", "f32"))
        page, slot = cache.place(torch.tensor([0], device="cuda"), torch.tensor([39], device="cuda"))
        good = out.clone()
        if where == "q":
            q[1, 2, 5] = math.nan
        elif fmt == "bf16":
            cache.pools["kv".index(where)][page, 1, slot, 3] = math.inf if where == "v" else math.nan
        else:
            cache.scales["kv".index(where)][page, 1, slot] = math.nan
        _attend(runtime, cache, lengths, q, 2, scale, out, ("f32", "f32"), 6)
        runtime.device_status()
        bad = torch.zeros_like(out, dtype=torch.bool)
        if where == "q":
            bad[1, 2] = True
        else:
            bad[1, 3:] = True  # the last token of sequence 0 sees position 39; heads 3 to 5 read key head 1
        touched = ~torch.isfinite(out)
        if where == "v" and fmt == "bf16":
            assert bool(touched[1, 3:, 3].all()) and not bool((touched & ~bad).any())
            bad[1, 3:] = touched[1, 3:]
        else:
            assert torch.equal(touched, bad)
        assert torch.equal(out[~bad], good[~bad])


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "bf16"])
def test_large_and_small_magnitudes(runtime, fmt):
    """Keys, values and queries of very different sizes from token to token; scores of hundreds."""
    import torch

    from attention_helpers import Cache, quantise64, POOLS, rounded

    lengths, heads, kv_heads, dim = [300, 77], 6, 2, 64
    cache = Cache(fmt, kv_heads, dim, 16, 2, 20)
    gen = torch.Generator(device="cuda").manual_seed(3)
    sequences = torch.cat([torch.full((n,), s, dtype=torch.int32) for s, n in enumerate(lengths)]).cuda()
    positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in lengths]).cuda()
    page, slot = cache.place(sequences, positions)
    for side in range(2):
        x = torch.randn(len(sequences), kv_heads, dim, generator=gen, device="cuda")
        size = torch.pow(10.0, torch.randint(-25, 26, (len(sequences), kv_heads, 1), generator=gen, device="cuda")) if side else 1.0
        codes, scales = quantise64(x * size, fmt)
        raw = torch.int16 if fmt == "bf16" else torch.uint8
        cache.pools[side].view(raw)[page, :, slot] = codes.to(POOLS[fmt]).view(raw)
        if scales is not None:
            cache.scales[side][page, :, slot] = scales
    for gain in (1e-30, 1e-3, 1.0, 40.0):
        q = gain * torch.randn(2, heads, dim, generator=gen, device="cuda")
        out = torch.full(q.shape, math.nan, device="cuda")
        # 40 times larger queries: scores of hundreds with a d of up to 2^-14 * 64 * 40 * 5 = 0.8 by the worst case; what counts
        # there is that the largest one wins: the scale of the test below is 1 / gain for them
        scale = dim ** -0.5 if gain <= 1 else dim ** -0.5 / gain
        _attend(runtime, cache, torch.tensor(lengths, dtype=torch.int32, device="cuda"), q, 1, scale, out, ("f32", "f32"), heads)
        runtime.device_status()
        from attention_helpers import attention64

        ref, bound = attention64(cache, lengths, q, 1, scale)
        assert bool(((out.double() - ref).abs() <= rounded(bound, ref, "f32")).all())


def test_one_score_far_above_the_others_takes_all(runtime):
    import torch

    from attention_helpers import Cache

    dim, n = 64, 500
    cache = Cache("bf16", 1, dim, 16, 1, 32)
    cache.pools[0].zero_()
    cache.pools[1].zero_()
    positions = torch.arange(n, dtype=torch.int32, device="cuda")
    page, slot = cache.place(torch.zeros_like(positions), positions)
    values = torch.randn(n, 1, dim, device="cuda").to(torch.bfloat16)
    cache.pools[1][page, :, slot] = values
    q = torch.zeros(1, 4, dim, device="cuda")
    q[0, :, 0] = torch.tensor([1e4, -1e4, 1e37, 1e4])
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    for at in (0, 17, 255, n - 1):
        cache.pools[0].zero_()
        cache.pools[0][page[at], 0, slot[at], 0] = 1.0
        _attend(runtime, cache, lengths, q, 1, 1.0, out, ("f32", "f32"), 4)
        runtime.device_status()
        assert torch.equal(out[0, 0], values[at, 0].float()) and torch.equal(out[0, 3], out[0, 0]) and torch.equal(out[0, 2], out[0, 0])
        others = torch.cat([values[:at], values[at + 1:]]).double().mean(0)[0]
        # 499 equal weights: each 16 bits of 1 exactly, the sum exact, values of size 4 summed in 32 bits
        assert float((out[0, 1].double() - others).abs().max()) < 1e-5


def test_equal_scores_give_the_mean(runtime):
    """Queries of zero: exact weights of 1."""
    import torch

    cache, lengths, q, out, scale = _case(runtime, "int8", [777], 1, 8, 2, 128, 16, ("f32", "f32"), check=False)
    q.zero_()
    _attend(runtime, cache, lengths, q, 1, scale, out, ("f32", "f32"), 8)
    runtime.device_status()
    at = torch.arange(777, dtype=torch.int32, device="cuda")
    v = cache.held(1, torch.zeros_like(at), at)[0]
    ref, size = v.mean(0).repeat_interleave(4, 0), v.abs().mean(0).repeat_interleave(4, 0)
    assert bool(((out[0].double() - ref).abs() <= 2.0 ** -16 * size).all())


@pytest.mark.parametrize("order", ["pth", "hpt", "thp"])
@pytest.mark.parametrize("fmt", ["int8", "bf16"])
def test_other_orders_and_gaps(runtime, fmt, order):
    _case(runtime, fmt, [100, 16, 45], 1, 12, 3, 48, 32, ("f32", "f32"), order=order, gap=16)


def test_keys_and_values_in_one_pool(runtime):
    """Pages that hold a key slab and a value slab, and a pool that is both."""
    import torch
    from dataclasses import replace

    from attention_helpers import Cache, attention64, rounded

    lengths, dim, kv_heads = [90, 33], 64, 2
    one = Cache("int8", 2 * kv_heads, dim, 16, 2, 6)  # heads 0, 1 are keys, 2, 3 values
    one.fill(lengths, 5)
    q = torch.randn(2, 6, dim, device="cuda")
    out = torch.empty_like(q)
    device_lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    halves = [one.scales[0][:, :kv_heads].contiguous(), one.scales[0][:, kv_heads:].contiguous()]
    for v_at, v_scales in ((kv_heads, halves[1]), (0, halves[0])):
        c = replace(one.c, kv_heads=kv_heads, v=one.c.k + v_at * one.stride["h"], k_scales=halves[0].data_ptr(), v_scales=v_scales.data_ptr())
        runtime.attention_device(c, one.t, device_lengths.data_ptr(), q.data_ptr(), 0, 6 * dim, 6, 1, 0.125, out.data_ptr(), 0, 6 * dim)
        runtime.device_status()
        two = Cache("int8", kv_heads, dim, 16, 2, 6)
        two.pools[0].copy_(one.pools[0][:, :kv_heads])
        two.pools[1].copy_(one.pools[0][:, v_at:v_at + kv_heads])
        two.scales = [halves[0], v_scales]
        ref, bound = attention64(two, lengths, q, 1, 0.125)
        assert bool(((out.double() - ref).abs() <= rounded(bound, ref, "f32")).all())


def test_shared_pages_and_strided_rows(runtime):
    """Sequences with the same pages (a common prefix); queries and outputs inside wider rows, whose other values stay."""
    import torch

    from attention_helpers import Cache, attention64, rounded, strided

    lengths, heads, kv_heads, dim, q_tokens = [64, 50, 7], 6, 3, 32, 2
    cache = Cache("int8", kv_heads, dim, 16, 3, 4, share=True)
    cache.fill([64, 0, 0], 4)
    width = heads * dim
    q_base, q = strided((6, width), width + 32, torch.float32, 3.0)
    q.normal_()
    out_base, out = strided((6 + 2, width), width + 8, torch.bfloat16, 5.0)
    _attend(runtime, cache, torch.tensor(lengths, dtype=torch.int32, device="cuda"), q_base, q_tokens, 0.2, out_base, ("f32", "bf16"), heads, width + 32, width + 8)
    runtime.device_status()
    ref, bound = attention64(cache, lengths, q.reshape(6, heads, dim), q_tokens, 0.2)
    got = out[:6].reshape(6, heads, dim).double()
    assert bool(((got - ref).abs() <= rounded(bound, ref, "bf16")).all())
    assert bool((out[6:] == 5.0).all()) and bool((out_base.view(8, -1)[:, width:] == 5.0).all())  # rows behind the last sequence


def test_pages_and_lengths_outside_are_reported(runtime):
    import torch

    from attention_helpers import attention64, rounded
    from qwen38_metal_b200 import Q4RuntimeError

    for bad_length, bad_page in ((-1, None), (129, None), ((1 << 31) - 1, None), (-(1 << 31), None), (None, -1), (None, 1 << 20)):
        cache, lengths, q, out, scale = _case(runtime, "int8", [60, 128], 1, 4, 2, 64, 16, ("f32", "f32"), per=8)
        good = out.clone()
        if bad_length is not None:
            lengths[1] = bad_length
        else:
            cache.table[1, 3] = bad_page
        _attend(runtime, cache, lengths, q, 1, scale, out, ("f32", "f32"), 4)
        with pytest.raises(Q4RuntimeError) as err:
            runtime.device_status()
        assert err.value.kind == "MappedTensorOutOfRange"
        runtime.device_status()
        ref, bound = attention64(cache, [60], q[:1], 1, scale)
        assert bool(((out[:1].double() - ref).abs() <= rounded(bound, ref, "f32")).all())
        if bad_length is not None and bad_length < 0:
            assert bool((out[1] == 0).all())
        elif bad_length is not None:
            # cut to the 128 tokens that the page table has
            ref, bound = attention64(cache, [60, 128], q, 1, scale)
            assert bool(((out.double() - ref).abs() <= rounded(bound, ref, "f32")).all())
        assert bool(out.isfinite().all())


def test_offsets_beyond_32_bits(runtime):
    """5 GB of keys; pages at both ends of them."""
    import torch

    from attention_helpers import Cache, attention64, rounded

    heads, dim, page, n = 4, 256, 64, 250
    pages = 5 * (1 << 30) // (heads * dim * page)
    cache = Cache("int8", heads, dim, page, 1, 4, spare=pages - 4, fill=0)
    cache.table[0] = torch.tensor([pages - 1, 0, pages // 2 + 1, pages - 2], dtype=torch.int32, device="cuda")
    cache.fill([n], 2)
    q = torch.randn(1, 24, dim, device="cuda")
    out = torch.empty_like(q)
    _attend(runtime, cache, torch.tensor([n], dtype=torch.int32, device="cuda"), q, 1, 0.0625, out, ("f32", "f32"), 24)
    runtime.device_status()
    ref, bound = attention64(cache, [n], q, 1, 0.0625)
    assert bool(((out.double() - ref).abs() <= rounded(bound, ref, "f32")).all())


def test_same_bits_every_time_and_in_graphs(runtime):
    """Two captured graphs and eager calls on one runtime, in turn; a graph follows lengths that change between replays."""
    import torch

    from attention_helpers import attention64, rounded

    a = _case(runtime, "int8", [9000, 40, 0, 3], 1, 24, 4, 256, 16, ("f32", "f32"), check=False)
    b = _case(runtime, "bf16", [700, 4000], 4, 8, 2, 64, 16, ("f32", "f32"), check=False)
    stream = torch.cuda.Stream()
    graphs = []
    for (cache, lengths, q, out, scale), q_tokens, heads in ((a, 1, 24), (b, 4, 8)):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            _attend(runtime, cache, lengths, q, q_tokens, scale, out, ("f32", "f32"), heads, stream=stream.cuda_stream)
        graphs.append(graph)
    first = [a[3].clone(), b[3].clone()]
    for _ in range(5):
        a[3].fill_(7.0)
        b[3].fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graphs[0].replay()
            graphs[1].replay()
        runtime.device_status()
        assert torch.equal(a[3], first[0]) and torch.equal(b[3], first[1])
    a[1].copy_(torch.tensor([17, 31, 5, 0], dtype=torch.int32))
    a[0].fill([17, 31, 5, 0], 9)
    torch.cuda.synchronize()
    graphs[0].replay()
    runtime.device_status()
    ref, bound = attention64(a[0], [17, 31, 5, 0], a[2], 1, a[4])
    assert bool(((a[3].double() - ref).abs() <= rounded(bound, ref, "f32")).all())


def test_calls_on_two_runtimes_at_once(runtime):
    """Each runtime has scratch of its own: calls on two streams, one runtime each, do not disturb one another."""
    import torch

    from qwen38_metal_b200 import CudaRuntime

    other = CudaRuntime(0)
    try:
        a = _case(runtime, "int8", [30000], 1, 24, 4, 256, 16, ("f32", "f32"), check=False)
        b = _case(other, "int8", [20000, 777], 1, 24, 4, 256, 16, ("f32", "f32"), seed=4, check=False)
        first = [a[3].clone(), b[3].clone()]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for _ in range(20):
            for rt, (cache, lengths, q, out, scale), s in ((runtime, a, streams[0]), (other, b, streams[1])):
                _attend(rt, cache, lengths, q, 1, scale, out, ("f32", "f32"), 24, stream=s.cuda_stream)
        runtime.device_status()
        other.device_status()
        assert torch.equal(a[3], first[0]) and torch.equal(b[3], first[1])
    finally:
        other.close()
