"""Rotary handles that have been closed are refused, also where none is a choice; the library is a stand-in here."""
import pytest


class _Library:
    def __getattr__(self, name):
        def call(*args):
            self.called.append(name)
            return 0

        return call

    def __init__(self):
        self.called = []


def _runtime():
    from qwen38_metal_b200 import CudaRuntime

    rt = CudaRuntime.__new__(CudaRuntime)
    rt._lib, rt._h = _Library(), None
    return rt


def _closed(rt):
    from qwen38_metal_b200 import Rotary

    rotary = Rotary(rt, object())
    rotary.close()
    rt._lib.called.clear()
    return rotary


def test_closed_handles_are_refused():
    from qwen38_metal_b200 import KvCache, KvTable, Q4RuntimeError

    rt = _runtime()
    cache, table = KvCache("int8", 1, 64, 16, 1, 16, 32, 48, 64), KvTable(16, 1, 1)
    write = lambda rotary: rt.kv_write_device(cache, table, 16, 0, 1, 16, 64, 32, 64, 0, rotary)  # noqa: E731
    turn = lambda rotary: rt.rotary_device(rotary, 16, 0, 64, 1, 1, 64, 16, 32, 0, 64)  # noqa: E731
    for call in (write, turn):
        with pytest.raises(Q4RuntimeError) as err:
            call(_closed(rt))
        assert err.value.kind == "InvalidArgument" and "closed" in str(err.value) and rt._lib.called == []
    write(None)
    assert rt._lib.called == ["q4b_kv_write_device"]
