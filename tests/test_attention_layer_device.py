"""What an attention layer refuses before it asks a GPU for anything: the runtime is a stand-in here."""
import pytest


class _Runtime:
    def __init__(self, device):
        self.device = device

    def rotary_create(self, *args, **kwargs):
        raise AssertionError("not reached")


def _jobs(heads, kv_heads, dim, hidden):
    from qwen38_metal_b200 import DeviceBuffer, MappedQ4AffineJob

    buffer = DeviceBuffer(0, 1 << 20)
    return [MappedQ4AffineJob(buffer, 0, buffer, 0, buffer, 0, rows) for rows in (heads * dim, kv_heads * dim, kv_heads * dim, hidden)]


class _Asked(Exception):
    pass


def _first_device(monkeypatch, **more):
    """The device that the layer's first buffer is asked for."""
    from qwen38_metal_b200 import attention

    def zeros(*shape, dtype=None, device=None):
        raise _Asked(device)

    monkeypatch.setattr(attention.torch, "zeros", zeros)
    with pytest.raises(_Asked) as asked:
        attention.AttentionLayer(_Runtime(more.pop("on")), *_jobs(4, 2, 64, 128), 128, 4, 2, 64, 1, 1, **more)
    return asked.value.args[0]


def test_buffers_are_on_the_runtimes_device(monkeypatch):
    import torch

    assert _first_device(monkeypatch, on=0) == torch.device("cuda", 0)
    assert _first_device(monkeypatch, on=1) == torch.device("cuda", 1)
    assert _first_device(monkeypatch, on=3, device=3) == torch.device("cuda", 3)


@pytest.mark.parametrize("on,device", [(0, 1), (1, 0), (2, 3)])
def test_another_device_than_the_runtimes_is_refused(monkeypatch, on, device):
    from qwen38_metal_b200 import Q4RuntimeError, attention

    monkeypatch.setattr(attention.torch, "zeros", lambda *a, **k: pytest.fail("memory asked for"))
    with pytest.raises(Q4RuntimeError) as err:
        attention.AttentionLayer(_Runtime(on), *_jobs(4, 2, 64, 128), 128, 4, 2, 64, 1, 1, device=device)
    assert err.value.kind == "InvalidArgument" and f"device {device}" in str(err.value)
