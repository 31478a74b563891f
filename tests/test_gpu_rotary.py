"""Rotary positions against the formula in 64 bits."""
import math

import pytest

pytestmark = pytest.mark.gpu

# fp32: cosine and sine are off by 2 units in the last place at most (2^-23) and by the rounding of the angle (2^-24 pi), the two
# products, their sum and the factor by 2^-24 each: less than 2^-21 (|a| + |b|)
SMALL = 2.0 ** -21


def _run(rt, x, positions, rotary, out, heads, dim, x_stride, out_stride, names, stream=0):
    from attention_helpers import kind

    rt.rotary_device(rotary, x.data_ptr(), kind(names[0]), x_stride, len(positions), heads, dim, positions.data_ptr(), out.data_ptr(), kind(names[1]), out_stride, stream)


def _check(got, x, positions, freq, factor, layout, name, exact=False):
    import torch

    from attention_helpers import rounded, turned64

    ref, size = turned64(x, positions, freq, factor, layout, exact)
    assert bool(((got.double() - ref).abs() <= rounded(SMALL * size, ref, name)).all())
    rest = 2 * len(freq)
    assert torch.equal(got[..., rest:], x[..., rest:].to(got.dtype))  # values that are not turned are only converted


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dim,rotary_dim", [(1, 24, 256, 64), (1, 1, 16, 16), (3, 5, 48, 6), (37, 3, 80, 80), (129, 24, 256, 256), (70, 4, 128, 98), (5, 7, 64, 2), (2, 4, 256, 254)])
@pytest.mark.parametrize("names", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
def test_against_formula(runtime, layout, tokens, heads, dim, rotary_dim, names):
    import torch

    from attention_helpers import DTYPES
    from qwen38_metal_b200 import rotary_frequencies

    gen = torch.Generator(device="cuda").manual_seed(tokens * dim)
    x = (3 * torch.randn(tokens, heads, dim, generator=gen, device="cuda")).to(DTYPES[names[0]])
    positions = torch.randint(0, 1 << 18, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    out = torch.full((tokens, heads, dim), math.nan, dtype=DTYPES[names[1]], device="cuda")
    rotary = runtime.rotary_create(rotary_dim, base=1e7, layout=layout)
    _run(runtime, x, positions, rotary, out, heads, dim, heads * dim, heads * dim, names)
    runtime.device_status()
    _check(out, x, positions, rotary_frequencies(rotary_dim, 1e7)[0], 1.0, layout, names[1])


@pytest.mark.parametrize("scaling", [{"kind": "linear", "factor": 4}, {"kind": "ntk", "factor": 8}, {"kind": "yarn", "factor": 4, "original_length": 65536}])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_far_positions_and_scaling(runtime, scaling, layout):
    """The smallest and largest positions that an int32 holds among them; negative ones turn the other way."""
    import torch

    from qwen38_metal_b200 import rotary_frequencies

    heads, dim, rotary_dim = 2, 128, 64
    positions = torch.tensor([0, 1, -1, 262143, 1 << 20, (1 << 31) - 1, -(1 << 31), 12345678], dtype=torch.int32, device="cuda")
    x = torch.randn(len(positions), heads, dim, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    out = torch.empty_like(x)
    rotary = runtime.rotary_create(rotary_dim, base=1e7, layout=layout, scaling=scaling)
    _run(runtime, x, positions, rotary, out, heads, dim, heads * dim, heads * dim, ("f32", "f32"))
    runtime.device_status()
    freq, factor = rotary_frequencies(rotary_dim, 1e7, scaling)
    _check(out, x, positions, freq, factor, layout, "f32", exact=True)
    assert torch.equal(out[0, :, rotary_dim:], x[0, :, rotary_dim:])


def test_own_frequencies_and_factor(runtime):
    import torch

    freq = [2.5, -0.75, 7.0, 0.0, 1e-9]
    x = torch.randn(40, 3, 32, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    positions = torch.arange(40, dtype=torch.int32, device="cuda") * 1001
    out = torch.empty_like(x)
    rotary = runtime.rotary_create(10, layout="half", inv_freq=freq, attention_factor=0.5)
    _run(runtime, x, positions, rotary, out, 3, 32, 96, 96, ("f32", "f32"))
    runtime.device_status()
    _check(out, x, positions, freq, 0.5, "half", "f32")


@pytest.mark.parametrize("names", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("heads,dim,rotary_dim", [(24, 256, 64), (3, 80, 80), (5, 48, 18)])
def test_in_place_and_strides(runtime, names, layout, heads, dim, rotary_dim):
    """In place inside wider rows; what lies between and behind the rows stays."""
    import torch

    from attention_helpers import DTYPES, strided
    from qwen38_metal_b200 import rotary_frequencies

    tokens, width, stride = 19, heads * dim, heads * dim + 64
    base, view = strided((tokens, width), stride, DTYPES[names[0]], 7.0)
    x = torch.randn(tokens, heads, dim, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda").to(DTYPES[names[0]])
    view.copy_(x.view(tokens, width))
    positions = torch.randint(0, 100000, (tokens,), device="cuda", dtype=torch.int32)
    rotary = runtime.rotary_create(rotary_dim, base=1e6, layout=layout)
    _run(runtime, base, positions, rotary, base, heads, dim, stride, stride, names)
    runtime.device_status()
    _check(view.reshape(tokens, heads, dim), x, positions, rotary_frequencies(rotary_dim, 1e6)[0], 1.0, layout, names[1])
    assert bool((base.view(tokens, stride)[:, width:] == 7.0).all())


def test_wrong_handles_are_refused(runtime):
    import torch

    from qwen38_metal_b200 import Q4RuntimeError

    x = torch.zeros(4, 32, device="cuda")
    positions = torch.zeros(4, dtype=torch.int32, device="cuda")
    rotary = runtime.rotary_create(64)
    with pytest.raises(Q4RuntimeError) as err:
        _run(runtime, x, positions, rotary, torch.empty_like(x), 1, 32, 32, 32, ("f32", "f32"))
    assert err.value.kind == "WrongLength"
    for bad in (dict(rotary_dim=63), dict(rotary_dim=0), dict(rotary_dim=64, layout="else"), dict(rotary_dim=8, inv_freq=[1.0])):
        with pytest.raises(Q4RuntimeError):
            runtime.rotary_create(**bad)


def test_other_stream_and_graph(runtime):
    import torch

    from qwen38_metal_b200 import rotary_frequencies

    x = torch.randn(300, 2, 64, device="cuda")
    positions = torch.arange(300, dtype=torch.int32, device="cuda")
    out, mid = torch.empty_like(x), torch.empty_like(x)
    rotary = runtime.rotary_create(64, base=1e5)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for _ in range(3):
            _run(runtime, x, positions, rotary, mid, 2, 64, 128, 128, ("f32", "f32"), stream.cuda_stream)
            out.copy_(mid)
    x.normal_()
    positions.add_(1000)
    torch.cuda.synchronize()
    graph.replay()
    runtime.device_status()
    _check(out, x, positions, rotary_frequencies(64, 1e5)[0], 1.0, "half", "f32")
