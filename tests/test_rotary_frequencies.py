"""Rotary frequencies and the refusals of the attention calls: host arithmetic, no GPU."""
import ctypes as C
import math

import numpy as np
import pytest


@pytest.fixture(scope="module")
def lib():
    from qwen38_metal_b200 import build, capi

    build.build()
    return capi.load()


def test_header_and_prototypes_agree(lib):
    import re

    from conftest import ROOT
    from qwen38_metal_b200 import capi

    text = re.sub(r"/\*.*?\*/", "", open(f"{ROOT}/include/q4b_attention.h").read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(q4b_[a-z0-9_]+)\s*\(", text)))
    assert names == sorted(capi.ATTENTION_EXPORTS)
    assert all(hasattr(lib, n) for n in names)
    assert C.sizeof(capi.Kv) == 80 and C.sizeof(capi.Table) == 24 and C.sizeof(capi.RotaryScaling) == 48


@pytest.mark.parametrize("dim", [2, 6, 64, 128, 256])
@pytest.mark.parametrize("base", [10000.0, 1e7])
def test_frequencies(dim, base):
    from qwen38_metal_b200 import rotary_frequencies

    i = np.arange(0, dim, 2) / dim
    freq, factor = rotary_frequencies(dim, base)
    # powers of two ways: a few units in the last place of 64 bits
    np.testing.assert_allclose(freq, base ** -i, rtol=1e-13)
    assert factor == 1.0
    freq, factor = rotary_frequencies(dim, base, {"kind": "linear", "factor": 4})
    np.testing.assert_allclose(freq, base ** -i / 4, rtol=1e-13)
    assert factor == 1.0
    freq, factor = rotary_frequencies(dim, base, {"kind": "ntk", "factor": 4})
    if dim > 2:  # the first pair keeps its frequency, the last one is stretched by the factor
        np.testing.assert_allclose(freq[[0, -1]], [1.0, base ** -i[-1] / 4], rtol=1e-12)
    assert factor == 1.0


@pytest.mark.parametrize("dim,base,original,factor", [(64, 1e7, 65536, 4.0), (128, 10000.0, 4096, 16.0), (128, 1e6, 32768, 1.5)])
def test_yarn(dim, base, original, factor):
    from qwen38_metal_b200 import rotary_frequencies

    plain, _ = rotary_frequencies(dim, base)
    freq, amplitude = rotary_frequencies(dim, base, {"kind": "yarn", "factor": factor, "original_length": original})
    turns = original * plain / (2 * math.pi)
    ratio = freq / plain
    assert amplitude == pytest.approx(0.1 * math.log(factor) + 1, rel=1e-14)
    assert np.all(np.diff(ratio) <= 1e-15) and np.all(ratio <= 1 + 1e-15) and np.all(ratio >= (1 - 1e-15) / factor)
    # the ramp's ends are rounded outwards to whole pairs
    low = np.nonzero(turns > 32)[0].max(initial=0)
    high = np.nonzero(turns < 1)[0].min(initial=dim // 2)
    np.testing.assert_allclose(ratio[:low + 1], 1.0, rtol=1e-14)
    np.testing.assert_allclose(ratio[high:], 1 / factor, rtol=1e-14)
    between = np.arange(low, min(high, dim // 2))
    # between them 1/ratio-weighted: ratio falls linearly in the pair's index
    np.testing.assert_allclose(np.diff(ratio[between], 2), 0.0, atol=1e-12)
    given = rotary_frequencies(dim, base, {"kind": "yarn", "factor": factor, "original_length": original, "fast_turns": 32,
                                           "slow_turns": 1, "attention_factor": 1.25})
    assert np.array_equal(given[0], freq) and given[1] == 1.25


@pytest.mark.parametrize("args,name", [
    ((0, 1e4, None), "EmptyDimension"), ((7, 1e4, None), "Unsupported"), ((258, 1e4, None), "Unsupported"),
    ((64, 1.0, None), "InvalidArgument"), ((64, math.nan, None), "InvalidArgument"), ((64, math.inf, None), "InvalidArgument"),
    ((64, 1e4, {"kind": "linear", "factor": 0}), "InvalidArgument"),
    ((64, 1e4, {"kind": "linear", "factor": math.inf}), "InvalidArgument"),
    ((64, 1e4, {"kind": "else", "factor": 2}), "InvalidArgument"),
    ((64, 1e4, {"kind": "yarn", "factor": 2}), "InvalidArgument"),
    ((64, 1e4, {"kind": "yarn", "factor": 2, "original_length": 4096, "fast_turns": 1, "slow_turns": 2}), "InvalidArgument"),
    ((64, 1e4, {"kind": "yarn", "factor": 2, "original_length": 4096, "attention_factor": -1}), "InvalidArgument"),
])
def test_frequency_refusals(lib, args, name):
    from qwen38_metal_b200 import Q4RuntimeError, rotary_frequencies

    with pytest.raises(Q4RuntimeError) as err:
        rotary_frequencies(*args)
    assert err.value.kind == name


# Addresses that nothing looks at: the checks of a call come before its runtime is asked for, and the last one says that there
# is none.
BIG = 1 << 32
K, V, KS, VS, TABLE, Q, OUT, POS, SEQ = (BIG * (i + 1) for i in range(9))


def _cache(**more):
    from qwen38_metal_b200 import KvCache

    return KvCache(**{**dict(format="int8", kv_heads=4, head_dim=256, page_tokens=16, pages=64, k=K, v=V, k_scales=KS, v_scales=VS), **more})


def _table(**more):
    from qwen38_metal_b200 import KvTable

    return KvTable(**{**dict(pages=TABLE, sequences=2, pages_per_sequence=8), **more})


def _status(lib, name, *args):
    from qwen38_metal_b200 import capi

    status = getattr(lib, name)(*args)
    return capi.STATUS_NAMES[status], lib.q4b_last_error().decode()


def _write(lib, cache=None, table=None, pos=POS, seq=SEQ, tokens=8, k=Q, k_stride=1024, v=OUT, v_stride=1024, dtype=0):
    return _status(lib, "q4b_kv_write_device", None, (cache or _cache()).c, (table or _table()).c, pos, seq, tokens, k, k_stride, v, v_stride, dtype, None, None)


def _read(lib, cache=None, table=None, pos=POS, seq=SEQ, tokens=8, k=Q, k_stride=1024, v=OUT, v_stride=1024, dtype=0):
    return _status(lib, "q4b_kv_read_device", None, (cache or _cache()).c, (table or _table()).c, pos, seq, tokens, k, k_stride, v, v_stride, dtype, None)


def _attend(lib, cache=None, table=None, lengths=POS, q=Q, q_dtype=0, q_stride=6144, heads=24, q_tokens=1, scale=0.0625, out=OUT, out_dtype=0, out_stride=6144):
    return _status(lib, "q4b_attention_device", None, (cache or _cache()).c, (table or _table()).c, lengths, q, q_dtype, q_stride, heads, q_tokens, scale, out, out_dtype,
                   out_stride, None)


NO_RUNTIME = ("InvalidArgument", "runtime handle is null")


def test_good_calls_get_as_far_as_the_runtime(lib):
    for call in (_write, _read, _attend):
        assert call(lib) == NO_RUNTIME
        assert call(lib, cache=_cache(format="bf16", k_scales=0, v_scales=0)) == NO_RUNTIME
        assert call(lib, cache=_cache(token_stride=1024, head_stride=256, page_stride=16384)) == NO_RUNTIME
        assert call(lib, cache=_cache(head_dim=16, token_stride=16, head_stride=512, page_stride=4096)) == NO_RUNTIME
        # keys and values side by side in one page
        assert call(lib, cache=_cache(v=K + 16384, token_stride=256, head_stride=4096, page_stride=32768)) == NO_RUNTIME
    for call in (_write, _read):
        assert call(lib, k=None) == NO_RUNTIME
        assert call(lib, v=None, cache=_cache(v=0, v_scales=0)) == NO_RUNTIME
        assert call(lib, seq=None) == NO_RUNTIME
        assert call(lib, v=Q + 4096, k_stride=2048, v_stride=2048) == NO_RUNTIME  # rows of keys and values


CACHES = [
    (dict(format="bf16", kv_heads=0), "EmptyDimension"), (dict(pages=0), "EmptyDimension"), (dict(page_tokens=0), "EmptyDimension"),
    (dict(head_dim=0), "EmptyDimension"), (dict(head_dim=100), "Unsupported"), (dict(head_dim=272), "Unsupported"), (dict(page_tokens=24), "Unsupported"),
    (dict(k=0), "InvalidArgument"), (dict(v=0), "InvalidArgument"), (dict(k_scales=0), "InvalidArgument"), (dict(v_scales=0), "InvalidArgument"),
    (dict(k=K + 8), "InvalidArgument"), (dict(v=V + 1), "InvalidArgument"), (dict(k_scales=KS + 4), "InvalidArgument"),
    (dict(token_stride=264, head_stride=8192, page_stride=65536), "InvalidArgument"),  # not a multiple of 16
    (dict(token_stride=240, head_stride=8192, page_stride=65536), "InvalidArgument"),  # shorter than a row
    (dict(token_stride=256, head_stride=2048, page_stride=65536), "InvalidArgument"),  # heads inside one another
    (dict(token_stride=256, head_stride=4096, page_stride=8192), "InvalidArgument"),
    (dict(token_stride=256, head_stride=4096, page_stride=1 << 41), "DimensionOverflow"),
    (dict(pages=1 << 31), "DimensionOverflow"),
]


@pytest.mark.parametrize("more,name", CACHES)
def test_cache_refusals(lib, more, name):
    for call in (_write, _read, _attend):
        got = call(lib, cache=_cache(**more))
        assert got[0] == name and got != NO_RUNTIME, got


@pytest.mark.parametrize("more,name", [
    (dict(pages=0), "InvalidArgument"), (dict(pages=TABLE + 2), "InvalidArgument"), (dict(sequences=0), "EmptyDimension"),
    (dict(pages_per_sequence=0), "EmptyDimension"), (dict(row_stride=7), "WrongLength"), (dict(pages_per_sequence=1 << 28), "DimensionOverflow"),
])
def test_table_refusals(lib, more, name):
    for call in (_write, _read, _attend):
        got = call(lib, table=_table(**more))
        assert got[0] == name and got != NO_RUNTIME, got


@pytest.mark.parametrize("more,name", [
    (dict(tokens=0), "EmptyDimension"), (dict(tokens=1 << 31), "DimensionOverflow"), (dict(pos=None), "InvalidArgument"), (dict(pos=POS + 2), "InvalidArgument"),
    (dict(k=None, v=None), "InvalidArgument"), (dict(k=Q + 8), "InvalidArgument"), (dict(k_stride=1026), "InvalidArgument"), (dict(k_stride=1020), "WrongLength"),
    (dict(dtype=2), "InvalidArgument"), (dict(seq=None, tokens=7), "WrongLength"), (dict(seq=SEQ + 1), "InvalidArgument"), (dict(k_stride=1 << 61), "DimensionOverflow"),
])
def test_token_refusals(lib, more, name):
    for call in (_write, _read):
        got = call(lib, **more)
        assert got[0] == name and got != NO_RUNTIME, got


@pytest.mark.parametrize("more,name", [
    (dict(heads=0), "EmptyDimension"), (dict(heads=22), "WrongLength"), (dict(q_tokens=0), "EmptyDimension"), (dict(q_tokens=17), "Unsupported"),
    (dict(scale=math.nan), "InvalidArgument"), (dict(scale=math.inf), "InvalidArgument"), (dict(lengths=None), "InvalidArgument"), (dict(q=None), "InvalidArgument"),
    (dict(out=None), "InvalidArgument"), (dict(q_dtype=5), "InvalidArgument"), (dict(out_dtype=-1), "InvalidArgument"), (dict(q_stride=6140), "WrongLength"),
    (dict(out_stride=6145), "InvalidArgument"), (dict(heads=65540), "DimensionOverflow"),
])
def test_attention_refusals(lib, more, name):
    got = _attend(lib, **more)
    assert got[0] == name and got != NO_RUNTIME, got


def test_more_tiles_than_32_bits_number_are_refused(lib):
    big = _table(sequences=1 << 16, pages_per_sequence=1 << 14)  # 2^30 tiles of four heads
    got = _attend(lib, table=big)
    assert got[0] == "DimensionOverflow" and "2^32" in got[1]
    assert _attend(lib, table=_table(sequences=(1 << 16) - 1, pages_per_sequence=1 << 14)) == NO_RUNTIME
    assert _attend(lib, table=_table(sequences=(1 << 16) - 1, pages_per_sequence=1 << 14), q_tokens=2)[0] == "DimensionOverflow"


def test_shared_memory_is_refused(lib):
    share = lambda got: got[0] == "InvalidArgument" and "share" in got[1]  # noqa: E731
    for at in (K, K + 64 * 4 * 16 * 256 - 16, V + 1024, KS, VS + 64):
        assert share(_attend(lib, out=at)) and share(_write(lib, k=at)) and share(_read(lib, v=at))
    assert share(_attend(lib, out=Q)) and share(_attend(lib, out=Q + 16)) and share(_attend(lib, out=POS)) and share(_attend(lib, out=TABLE))
    assert share(_read(lib, k=Q, v=Q)) and share(_read(lib, k=Q, v=Q + 1024, k_stride=2048, v_stride=2048))
    assert share(_read(lib, k=POS)) and share(_read(lib, v=TABLE)) and share(_write(lib, cache=_cache(v=K)))
    assert share(_write(lib, table=_table(pages=KS)))
    assert _attend(lib, cache=_cache(v=K)) == NO_RUNTIME  # reading one pool as both is allowed


def test_one_token_has_no_step_from_one_row_to_the_next(lib):
    share = lambda got: got[0] == "InvalidArgument" and "share" in got[1]  # noqa: E731
    one = dict(tokens=1, k_stride=0, v_stride=0)
    assert _read(lib, **one) == NO_RUNTIME and _write(lib, **one) == NO_RUNTIME
    assert share(_read(lib, k=Q, v=Q, **one)) and share(_read(lib, k=Q, v=Q + 16, **one)) and share(_read(lib, k=Q + 4080, v=Q, **one))
    assert _read(lib, k=Q, v=Q + 4096, **one) == NO_RUNTIME


def test_keys_and_values_that_would_be_written_over_each_other_are_refused(lib):
    share = lambda got: got[0] == "InvalidArgument" and "share" in got[1]  # noqa: E731
    page = 4 * 16 * 256
    for off in (16, 240, 256, 4096, page, 63 * page + 16, 64 * page - 256):
        assert share(_write(lib, cache=_cache(v=K + off))) and share(_write(lib, cache=_cache(k=V + off))), off
    assert _write(lib, cache=_cache(v=K + 64 * page)) == NO_RUNTIME
    # pages of keys, then of values; heads of both in turn; rows of both in turn
    for strides, off in ((dict(token_stride=256, head_stride=4096, page_stride=2 * page), page), (dict(token_stride=256, head_stride=8192, page_stride=2 * page), 4096),
                         (dict(token_stride=512, head_stride=8192, page_stride=2 * page), 256), (dict(token_stride=2048, head_stride=512, page_stride=2 * page), 256)):
        assert _write(lib, cache=_cache(v=K + off, **strides)) == NO_RUNTIME
        assert _write(lib, cache=_cache(k=V + off, **strides)) == NO_RUNTIME
        assert _write(lib, cache=_cache(v=K + off + 2 * page, **strides)) == NO_RUNTIME
        assert share(_write(lib, cache=_cache(v=K + off - 16, **strides))) and share(_write(lib, cache=_cache(v=K + off + 2 * page + 240, **strides)))
    assert share(_write(lib, cache=_cache(v_scales=KS))) and share(_write(lib, cache=_cache(v_scales=KS + 16)))
    assert _write(lib, k=None, cache=_cache(k=V + 16, k_scales=VS)) == NO_RUNTIME  # one side alone


def test_rotary_refusals(lib):
    def call(rotary=None, x=Q, x_dtype=0, x_stride=6144, tokens=4, heads=24, head_dim=256, pos=POS, out=OUT, out_dtype=0, out_stride=6144):
        return _status(lib, "q4b_rotary_device", None, rotary, x, x_dtype, x_stride, tokens, heads, head_dim, pos, out, out_dtype, out_stride, None)

    no_handle = ("InvalidArgument", "rotary handle is null")
    assert call() == no_handle and call(out=Q) == no_handle and call(out=Q, tokens=1, out_stride=8192) == no_handle
    for more, name in ((dict(tokens=0), "EmptyDimension"), (dict(heads=0), "EmptyDimension"), (dict(head_dim=0), "EmptyDimension"), (dict(head_dim=100), "Unsupported"),
                       (dict(head_dim=512), "Unsupported"), (dict(heads=1 << 17), "DimensionOverflow"), (dict(tokens=1 << 31), "DimensionOverflow"), (dict(x=None), "InvalidArgument"),
                       (dict(out=None), "InvalidArgument"), (dict(pos=None), "InvalidArgument"), (dict(x=Q + 4), "InvalidArgument"), (dict(out_stride=6146), "InvalidArgument"),
                       (dict(x_stride=4096), "WrongLength"), (dict(x_dtype=7), "InvalidArgument"), (dict(out=Q, out_dtype=1), "InvalidArgument"),
                       (dict(out=Q, out_stride=8192), "InvalidArgument"), (dict(out=Q + 16), "InvalidArgument"), (dict(out=POS - 64), "InvalidArgument")):
        got = call(**more)
        assert got[0] == name and got != no_handle, (more, got)
    freq, out = (C.c_double * 4)(1.0, 0.5, 0.25, math.nan), C.c_void_p()
    create = lambda *a: _status(lib, "q4b_rotary_create", None, *a)  # noqa: E731
    assert create(freq, 8, 0, 1.0, None)[0] == "InvalidArgument"
    assert create(None, 8, 0, 1.0, C.byref(out))[0] == "InvalidArgument"
    assert "not finite" in create(freq, 8, 0, 1.0, C.byref(out))[1]
    assert create(freq, 6, 0, 1.0, C.byref(out)) == NO_RUNTIME
    assert create(freq, 6, 2, 1.0, C.byref(out))[0] == "InvalidArgument"
    assert create(freq, 6, 0, math.inf, C.byref(out))[0] == "InvalidArgument"
    assert create(freq, 0, 0, 1.0, C.byref(out))[0] == "EmptyDimension"
    assert create(freq, 5, 0, 1.0, C.byref(out))[0] == "Unsupported"
    lib.q4b_rotary_destroy(None)
