"""The short host path of the 8-bit products, without a GPU: torch without its private functions, another current device."""
import contextlib
import importlib.util

import torch


def copy_of_ops():
    import tmq_b200.ops as ops
    spec = importlib.util.spec_from_file_location("tmq_b200.ops_once_more", ops.__file__)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_without_torchs_private_functions(monkeypatch):
    monkeypatch.delattr(torch._C, "_cuda_getDevice", raising=False)
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    ops = copy_of_ops()

    class Stream:
        def __init__(self, index):
            self.cuda_stream = 1000 + index

    monkeypatch.setattr(torch.cuda, "current_stream", Stream)
    assert ops._current_device is torch.cuda.current_device
    assert ops._raw_stream(3) == 1003


def test_a_call_on_a_device_that_is_not_current(monkeypatch):
    from tmq_b200 import ops
    entered = []

    @contextlib.contextmanager
    def device(index):
        entered.append(index)
        yield
        entered.append("left")

    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", device)
    call = lambda *args: (args, list(entered))
    assert ops._enqueue(call, 0, (1, 2)) == ((1, 2), []) and entered == []
    assert ops._enqueue(call, 1, (3,)) == ((3,), [1]) and entered == [1, "left"]
