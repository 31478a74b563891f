"""Index arithmetic of the cache and attention kernels at the ends of the sizes that their calls accept, on the CPU."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest

from conftest import ROOT


@pytest.fixture(scope="module")
def shim():
    out = os.path.join(tempfile.mkdtemp(prefix="attention_index"), "shim.so")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", out, os.path.join(ROOT, "tests", "attention_index_shim.cpp")])
    lib = C.CDLL(out)
    lib.shim_kv_scale_index.restype = C.c_uint64
    lib.shim_kv_scale_index.argtypes = [C.c_uint64, C.c_uint32, C.c_uint32]
    lib.shim_attention_hidden.argtypes = [C.c_int32, C.c_int32, C.c_int32]
    return lib


@pytest.mark.parametrize("kv_heads,page_tokens,page", [(1, 16, 0), (4, 16, 1000), (8, 1 << 20, 3), (4096, 1 << 20, 1), (65535, 1 << 20, 7), (65535, 65552, 2)])
def test_scales_of_all_heads(shim, kv_heads, page_tokens, page):
    """[page][head][token of the page] without gaps, beyond 32 bits within one page too."""
    for head in {0, kv_heads // 2, kv_heads - 1}:
        for slot in (0, page_tokens - 1):
            first = page * kv_heads * page_tokens + slot
            assert shim.shim_kv_scale_index(first, head, page_tokens) == (page * kv_heads + head) * page_tokens + slot


@pytest.mark.parametrize("tokens", [16, 32])
@pytest.mark.parametrize("sure", [-15, 0, 1, 15, 16, 17, 1000, (1 << 31) - 16, (1 << 31) - 17, (1 << 31) - 31, (1 << 31) - 33])
def test_tokens_that_some_rows_do_not_see(shim, tokens, sure):
    """Steps of 16 tokens up to the end of the longest page table, 2^31 - 16 tokens."""
    last = (1 << 31) - 32
    for token in {0, 16, last, last - 16, last - 32, last - 48, max(sure // 16 * 16, 0), max(sure // 16 * 16 - tokens, 0), min(max(sure // 16 * 16 + 16, 0), last)}:
        if 0 <= token <= last:
            assert bool(shim.shim_attention_hidden(token, tokens, sure)) == (token + tokens > sure), token
