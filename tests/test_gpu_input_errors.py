"""Reports of what only the device can see: each call's own, whatever was reported and taken back just before, on any stream."""
import pytest

pytestmark = pytest.mark.gpu


def test_every_call_that_meets_a_bad_page_is_reported(runtime):
    import torch

    from attention_helpers import Cache, kind
    from qwen38_metal_b200 import Q4RuntimeError

    dim, heads, n = 64, 4, 40
    good, bad = (Cache("int8", 2, dim, 16, 1, 3, seed=s) for s in (1, 2))
    for cache in (good, bad):
        cache.fill([n], 1)
    bad.table[0, 1] = bad.pages
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    q, out = torch.randn(1, heads, dim, device="cuda"), torch.empty(1, heads, dim, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(60):
        cache = (bad, bad, good)[i % 3]
        runtime.attention_device(cache.c, cache.t, lengths.data_ptr(), q.data_ptr(), kind("f32"), heads * dim, heads, 1, 0.125, out.data_ptr(), kind("f32"),
                                 heads * dim, streams[i % 2].cuda_stream)
        if cache is good:
            runtime.device_status()
            continue
        with pytest.raises(Q4RuntimeError) as err:
            runtime.device_status()
        assert err.value.kind == "MappedTensorOutOfRange"
