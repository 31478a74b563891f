"""The paged cache: codes and scales are those of the definition to the last bit, rows that are not written stay."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _write(rt, cache, positions, sequences, k, v, name, rotary=None, stream=0, k_stride=None, v_stride=None):
    from attention_helpers import kind

    width = cache.kv_heads * cache.dim
    rt.kv_write_device(cache.c, cache.t, positions.data_ptr(), sequences.data_ptr() if sequences is not None else 0, len(positions), k.data_ptr() if k is not None else 0,
                       k_stride or width, v.data_ptr() if v is not None else 0, v_stride or width, kind(name), rotary, stream)


def _read(rt, cache, positions, sequences, k, v, name, stream=0, k_stride=None, v_stride=None):
    from attention_helpers import kind

    width = cache.kv_heads * cache.dim
    rt.kv_read_device(cache.c, cache.t, positions.data_ptr(), sequences.data_ptr() if sequences is not None else 0, len(positions), k.data_ptr() if k is not None else 0,
                      k_stride or width, v.data_ptr() if v is not None else 0, v_stride or width, kind(name), stream)


def _inputs(tokens, heads, dim, name, seed):
    import torch

    from attention_helpers import DTYPES

    gen = torch.Generator(device="cuda").manual_seed(seed)
    size = torch.exp(3 * torch.randn(tokens, heads, 1, generator=gen, device="cuda"))
    return [(size * torch.randn(tokens, heads, dim, generator=gen, device="cuda")).to(DTYPES[name]) for _ in range(2)]


def _check_held(cache, side, sequences, positions, x):
    import torch

    from attention_helpers import POOLS, quantise64

    codes, scales = quantise64(x, cache.fmt)
    _, raw, held = cache.held(side, sequences, positions)
    got = raw.view(POOLS[cache.fmt]).float()
    assert torch.equal(torch.where(got == 0, 0.0, got), torch.where(codes == 0, 0.0, codes.float()))
    if scales is not None:
        assert torch.equal(torch.nan_to_num(held, nan=-1.0), torch.nan_to_num(scales, nan=-1.0))
    return codes, scales


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "bf16"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("heads,dim,page,lengths", [(4, 256, 16, [1]), (4, 256, 16, [16, 17, 1]), (1, 16, 16, [40, 3]), (3, 80, 48, [97, 48]), (8, 128, 64, [65, 1, 200]), (2, 192, 32, [31]),
                                                   (5, 64, 256, [300])])
def test_written_and_read_back(runtime, fmt, name, heads, dim, page, lengths):
    import torch

    from attention_helpers import DTYPES, Cache

    per = max((n + page - 1) // page for n in lengths)
    cache = Cache(fmt, heads, dim, page, len(lengths), per)
    before = [r.clone() for r in cache.raw]
    sequences = torch.cat([torch.full((n,), s, dtype=torch.int32) for s, n in enumerate(lengths)]).cuda()
    positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in lengths]).cuda()
    order = torch.randperm(len(positions), device="cuda")
    sequences, positions = sequences[order].contiguous(), positions[order].contiguous()
    k, v = _inputs(len(positions), heads, dim, name, dim)
    _write(runtime, cache, positions, sequences, k, v, name)
    runtime.device_status()
    for side, x in ((0, k), (1, v)):
        codes, scales = _check_held(cache, side, sequences, positions, x)
        # what no token was written to is as it was
        page_at, slot = cache.place(sequences, positions)
        untouched = torch.ones(cache.pages, page, dtype=torch.bool, device="cuda")
        untouched[page_at, slot] = False
        rows = cache.raw[side].view(cache.pages, heads, page, -1).transpose(1, 2)[untouched]
        assert torch.equal(rows, before[side].view(cache.pages, heads, page, -1).transpose(1, 2)[untouched])
        if scales is not None:
            assert bool(cache.scales[side].transpose(1, 2)[untouched].isnan().all())
    for out_name in ("f32", "bf16"):
        out = [torch.full(k.shape, 5.0, dtype=DTYPES[out_name], device="cuda") for _ in range(2)]
        _read(runtime, cache, positions, sequences, out[0], out[1], out_name)
        runtime.device_status()
        for side, x in ((0, k), (1, v)):
            held = cache.held(side, sequences, positions)
            ref = (held[0] if held[2] is None else held[0]).float().to(DTYPES[out_name])
            assert torch.equal(out[side], ref)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_codes_on_and_next_to_borders(runtime, fmt):
    """Values at the middle between two codes, and one unit in the last place to either side, for scales of every size."""
    import torch

    from attention_helpers import TOP, Cache

    dim, heads = 256, 1
    scales = [1.0, 0.1, 1 / 3, 3e-5, 7e8, 2.0 ** -99, 2.0 ** -101, 1.7e-38, 3e-43, 1e33]
    rows = []
    for s in scales:
        amax = torch.tensor(TOP[fmt] * s, dtype=torch.float64).float()
        scale = (amax.double() / TOP[fmt]).float()
        if fmt == "int8":
            middles = torch.arange(-126.5, 127.0, 4.0)
        else:
            codes = torch.arange(128, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).float()[:-1]
            middles = ((codes[1:] + codes[:-1]) / 2)[::2]
        x = (middles.double() * scale.double()).float()
        row = torch.cat([amax[None], x, torch.nextafter(x, torch.tensor(math.inf)), torch.nextafter(x, torch.tensor(-math.inf))])[:dim]
        rows.append(torch.nn.functional.pad(row, (0, dim - len(row))))
    x = torch.stack(rows)[:, None].cuda().contiguous()
    assert bool((x.abs().amax(-1) == x[..., 0].abs()).all())
    cache = Cache(fmt, heads, dim, 16, 1, 1)
    positions, sequences = torch.arange(len(scales), dtype=torch.int32, device="cuda"), torch.zeros(len(scales), dtype=torch.int32, device="cuda")
    _write(runtime, cache, positions, sequences, x, -x, "f32")
    runtime.device_status()
    _check_held(cache, 0, sequences, positions, x)
    _check_held(cache, 1, sequences, positions, -x)


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "bf16"])
def test_zero_rows_and_numbers_that_are_not_finite(runtime, fmt):
    import torch

    from attention_helpers import Cache

    dim = 64
    x = torch.randn(6, 1, dim, device="cuda")
    x[0] = 0.0
    x[1, 0, 7] = math.nan
    x[2, 0, 9] = math.inf
    x[3, 0, 63] = -math.inf
    x[4] = 1e-45
    cache = Cache(fmt, 1, dim, 16, 1, 1)
    positions, sequences = torch.arange(6, dtype=torch.int32, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    _write(runtime, cache, positions, sequences, x, x, "f32")
    out = torch.full((2, 6, 1, dim), 5.0, device="cuda")
    _read(runtime, cache, positions, sequences, out[0], out[1], "f32")
    runtime.device_status()
    for o in out:
        assert bool((o[0] == 0).all()) and bool(o[5].isfinite().all())
        if fmt == "bf16":
            assert bool(o[1, 0, 7].isnan()) and o[2, 0, 9] == math.inf and o[3, 0, 63] == -math.inf and int(o[1:4].isfinite().logical_not().sum()) == 3
        else:
            assert bool(o[1:4].isnan().all()) and bool((o[4] == 0).all())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("fmt,name,dim,rotary_dim", [("int8", "f32", 256, 64), ("e4m3", "bf16", 128, 128), ("bf16", "f32", 80, 78), ("int8", "bf16", 48, 6)])
def test_keys_turned_on_the_way(runtime, fmt, name, dim, rotary_dim, layout):
    import torch

    from attention_helpers import TOP, Cache, turned64
    from qwen38_metal_b200 import rotary_frequencies

    tokens, heads = 50, 3
    cache = Cache(fmt, heads, dim, 16, 1, 7)
    positions = torch.arange(3, 3 + tokens, dtype=torch.int32, device="cuda")
    sequences = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    k, v = _inputs(tokens, heads, dim, name, 3)
    rotary = runtime.rotary_create(rotary_dim, base=1e6, layout=layout)
    _write(runtime, cache, positions, sequences, k, v, name, rotary)
    runtime.device_status()
    _check_held(cache, 1, sequences, positions, v)  # values are not turned
    ref, size = turned64(k, positions, rotary_frequencies(rotary_dim, 1e6)[0], 1.0, layout)
    got, raw, scales = cache.held(0, sequences, positions)
    # 2^-21 (|a| + |b|) for the turn; half a step of the code: of a whole number 0.5, of e4m3 2^-4 of the value or 2^-10 below its
    # normal numbers; the scale itself is off by what the row's largest value is, 2^-21 of its pair, and its rounding 2^-24
    worst = size.amax(-1, keepdim=True).clamp(min=1e-30) + ref.abs().amax(-1, keepdim=True)
    if fmt == "bf16":
        bound = 2.0 ** -21 * size + 2.0 ** -8 * (ref.abs() + 2.0 ** -21 * size)
    elif fmt == "int8":
        bound = 2.0 ** -20 * worst + 0.5001 * scales.double()[..., None]
    else:
        bound = 2.0 ** -20 * worst + torch.maximum(2.0 ** -4 * ref.abs() * 1.001, 2.0 ** -10 * 1.001 * scales.double()[..., None])
    assert bool(((got - ref).abs() <= bound).all())
    if scales is not None:
        amax = ref.abs().amax(-1)
        assert bool(((scales.double() * TOP[fmt] - amax).abs() <= 2.0 ** -20 * worst[..., 0]).all())


@pytest.mark.parametrize("order", ["pth", "hpt", "thp"])
@pytest.mark.parametrize("fmt", ["int8", "bf16"])
def test_other_orders_and_gaps(runtime, fmt, order):
    """Heads inside tokens, heads outside pages, pages inside tokens, with gaps; rows of activations with gaps."""
    import torch

    from attention_helpers import Cache, strided

    heads, dim, page = 3, 48, 32
    cache = Cache(fmt, heads, dim, page, 2, 3, order=order, gap=16)
    raw_before = [r.clone() for r in cache.raw]
    lengths = [70, 33]
    sequences = torch.cat([torch.full((n,), s, dtype=torch.int32) for s, n in enumerate(lengths)]).cuda()
    positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in lengths]).cuda()
    tokens, width = len(positions), heads * dim
    # keys and values beside each other in rows, as one projection leaves them
    base, rows = strided((tokens, 2 * width), 2 * width + 16, torch.float32, 9.0)
    rows.normal_()
    k, v = (rows[:, i * width:(i + 1) * width] for i in range(2))
    _write(runtime, cache, positions, sequences, k, v, "f32", k_stride=2 * width + 16, v_stride=2 * width + 16)
    back, back_rows = strided((tokens, 2 * width), 2 * width + 16, torch.float32, 9.0)
    _read(runtime, cache, positions, sequences, back_rows, back_rows[:, width:], "f32", k_stride=2 * width + 16, v_stride=2 * width + 16)
    runtime.device_status()
    for side, x in ((0, k), (1, v)):
        _check_held(cache, side, sequences, positions, x.reshape(tokens, heads, dim))
        assert torch.equal(back_rows[:, side * width:(side + 1) * width].reshape(tokens, heads, dim), cache.held(side, sequences, positions)[0].float())
        # gaps keep their bytes: put back what the rows held before and compare all memory
        changed = cache.raw[side].clone()
        view = torch.as_strided(changed.view(cache.pools[side].dtype), cache.pools[side].shape, cache.pools[side].stride())
        old = torch.as_strided(raw_before[side].view(cache.pools[side].dtype), cache.pools[side].shape, cache.pools[side].stride())
        raw_type = torch.int16 if fmt == "bf16" else torch.uint8
        view.view(raw_type).copy_(old.view(raw_type))
        assert torch.equal(changed, raw_before[side])
    assert bool((back.view(tokens, -1)[:, 2 * width:] == 9.0).all())


def test_one_side_and_runs_without_sequences(runtime):
    import torch

    from attention_helpers import Cache

    heads, dim, each = 2, 64, 5
    cache = Cache("int8", heads, dim, 16, 3, 2)
    positions = torch.tensor([0, 1, 2, 3, 4, 10, 11, 12, 13, 14, 27, 28, 29, 30, 31], dtype=torch.int32, device="cuda")
    sequences = torch.arange(3, dtype=torch.int32, device="cuda").repeat_interleave(each)
    k, v = _inputs(15, heads, dim, "f32", 4)
    _write(runtime, cache, positions, None, k, None, "f32")
    runtime.device_status()
    _check_held(cache, 0, sequences, positions, k)
    assert bool((cache.raw[1] == 0xff).all()) and bool(cache.scales[1].isnan().all())
    _write(runtime, cache, positions, None, None, v, "f32")
    _check_held(cache, 0, sequences, positions, k)
    _check_held(cache, 1, sequences, positions, v)
    out = torch.full(k.shape, 5.0, device="cuda")
    _read(runtime, cache, positions, None, None, out, "f32")
    runtime.device_status()
    assert torch.equal(out, cache.held(1, sequences, positions)[0].float())


@pytest.mark.parametrize("tokens", [40, 3000])
def test_last_of_equal_places_is_kept_and_padded_tokens_are_left_out(runtime, tokens):
    import torch

    from attention_helpers import Cache

    heads, dim, sequences_n = 2, 32, 3
    cache = Cache("int8", heads, dim, 16, sequences_n, 4)
    gen = torch.Generator().manual_seed(tokens)
    positions = torch.randint(-3, 60, (tokens,), generator=gen, dtype=torch.int32)
    sequences = torch.randint(0, sequences_n, (tokens,), generator=gen, dtype=torch.int32)
    positions[0] = -(1 << 31)
    sequences[0] = -5  # of a padded token: nobody looks
    last = {}
    for t, (s, p) in enumerate(zip(sequences.tolist(), positions.tolist())):
        if p >= 0:
            last[(s, p)] = t
    keep = torch.tensor(sorted(last.values()))
    k, v = _inputs(tokens, heads, dim, "f32", 8)
    positions, sequences = positions.cuda(), sequences.cuda()
    results = []
    for _ in range(2):
        cache.raw[0].fill_(0)
        cache.raw[1].fill_(0)
        _write(runtime, cache, positions, sequences, k, v, "f32")
        runtime.device_status()
        for side, x in ((0, k), (1, v)):
            _check_held(cache, side, sequences[keep], positions[keep], x[keep])
        results.append([r.clone() for r in cache.raw])
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    out = torch.full((2,) + k.shape, 5.0, device="cuda")
    _read(runtime, cache, positions, sequences, out[0], out[1], "f32")
    runtime.device_status()
    padded = positions < 0
    assert bool(padded.any()) and bool((out[:, padded] == 5.0).all())
    assert torch.equal(out[0][~padded], cache.held(0, sequences[~padded], positions[~padded])[0].float())


def test_places_outside_are_left_out_and_reported(runtime):
    """Sequence numbers, positions and page numbers that do not exist; their tokens touch nothing, the others are right."""
    import torch

    from attention_helpers import Cache
    from qwen38_metal_b200 import Q4RuntimeError

    heads, dim = 2, 32
    good_s, good_p = [0, 1, 1], [3, 0, 31]
    for bad_s, bad_p, bad_page in ((2, 0, None), (-1, 0, None), (0, 32, None), (1, (1 << 31) - 1, None), (0, 20, 1 << 20), (0, 20, -1), (0, 20, 6)):
        cache = Cache("int8", heads, dim, 16, 2, 2, spare=2)
        assert cache.pages == 6
        if bad_page is not None:
            cache.table[0, 1] = bad_page
        before = [r.clone() for r in cache.raw]
        s = torch.tensor(good_s + [bad_s], dtype=torch.int32, device="cuda")
        p = torch.tensor(good_p + [bad_p], dtype=torch.int32, device="cuda")
        k, v = _inputs(4, heads, dim, "f32", 9)
        _write(runtime, cache, p, s, k, v, "f32")
        with pytest.raises(Q4RuntimeError) as err:
            runtime.device_status()
        assert err.value.kind == "MappedTensorOutOfRange"
        runtime.device_status()  # told once
        _check_held(cache, 0, s[:3], p[:3], k[:3])
        changed = (cache.raw[0] != before[0]).view(cache.pages, heads, 16, dim).any(-1).any(1)
        assert int(changed.sum()) <= 3
        out = torch.full(k.shape, 5.0, device="cuda")
        _read(runtime, cache, p, s, out, None, "f32")
        with pytest.raises(Q4RuntimeError):
            runtime.device_status()
        assert bool((out[3] == 5.0).all()) and torch.equal(out[:3], cache.held(0, s[:3], p[:3])[0].float())


def test_offsets_beyond_32_bits(runtime):
    """A pool of 5 GB: first and last pages."""
    import torch

    from attention_helpers import Cache

    heads, dim, page = 4, 256, 64
    pages = 5 * (1 << 30) // (heads * dim * page)
    cache = Cache("int8", heads, dim, page, 1, 4, spare=pages - 4)
    assert cache.raw[0].numel() > 5 * (1 << 30) - (1 << 20)
    cache.table[0] = torch.tensor([pages - 1, 0, pages // 2 + 1, pages - 2], dtype=torch.int32, device="cuda")
    positions = torch.tensor([0, 63, 64, 127, 128, 255], dtype=torch.int32, device="cuda")
    sequences = torch.zeros(6, dtype=torch.int32, device="cuda")
    k, v = _inputs(6, heads, dim, "f32", 10)
    _write(runtime, cache, positions, sequences, k, v, "f32")
    out = torch.zeros(2, 6, heads, dim, device="cuda")
    _read(runtime, cache, positions, sequences, out[0], out[1], "f32")
    runtime.device_status()
    for side, x in ((0, k), (1, v)):
        _check_held(cache, side, sequences, positions, x)
        assert torch.equal(out[side], cache.held(side, sequences, positions)[0].float())
