"""B200 (sm_100a) implementation of the affine-Q4 projection path of Fuxx-1/qwen38-metal.

All compute lives in `lib/libq4b200.so` (CUDA, built by `qwen38_metal_b200.build`); this package is the
host-side mirror of the reference's projection interface over that library's C ABI
(`include/q4b200.h`), and of the attention calls that stand between projections (`include/q4b_attention.h`). There is no CPU or PyTorch compute path: without the library, or without a
B200, constructing a runtime raises.
"""
from .runtime import (CudaRuntime, DeviceBuffer, KvCache, KvTable, MappedQ4AffineJob, Q4RuntimeError, Rotary,  # noqa: F401
                      rotary_frequencies)

__all__ = ["AttentionLayer", "CudaRuntime", "DeviceBuffer", "KvCache", "KvTable", "MappedQ4AffineJob", "Q4RuntimeError", "Rotary",
           "rotary_frequencies"]


def __getattr__(name):  # (needs torch, which the calls over host buffers do not)
    if name == "AttentionLayer":
        from .attention import AttentionLayer

        return AttentionLayer
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
