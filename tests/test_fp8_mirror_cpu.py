"""The Python mirror of the 8-bit operators and the grouped router, without a GPU: what it asks torch for, and the calls it refuses before the library sees them."""
import pytest
import torch

from eke_hive_b200 import ops


def test_streams_and_memory_without_torchs_private_names(monkeypatch):
    asked = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: type("S", (), {"cuda_stream": 70 + d})())
    monkeypatch.setattr(torch, "empty_strided", lambda size, stride, dtype, device: asked.append((size, stride, dtype, device)))
    monkeypatch.setattr(ops, "_raw_stream", None)
    assert ops._stream() == 73 and ops._stream(1) == 71
    for name in ("_empty_cuda", "_dispatch_modes"):
        with monkeypatch.context() as m:
            m.setattr(ops, name, None)
            asked.clear()
            ops._empty(5, 7, torch.int32)
            ops._bytes(9)
            assert asked == [((5, 7), (7, 1), torch.int32, "cuda"), ((9,), (1,), torch.uint8, "cuda")]


def test_memory_is_allocated_where_modes_see_it(monkeypatch):
    """Under a dispatch mode, and where uninitialised memory may have to be filled, an allocation goes through torch's dispatcher."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    public, private = [], []
    monkeypatch.setattr(torch, "empty_strided", lambda *a, **k: public.append(a))
    monkeypatch.setattr(ops, "_empty_cuda", lambda *a: private.append(a))
    monkeypatch.setattr(ops, "_dispatch_modes", torch._C._len_torch_dispatch_stack)
    ops._empty(2, 3, torch.float32)
    assert (len(public), len(private)) == (0, 1)
    with Mode():
        ops._empty(2, 3, torch.float32)
        ops._bytes(4)
    assert (len(public), len(private)) == (2, 1)
    was = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)
    try:
        ops._bytes(4)
    finally:
        torch.use_deterministic_algorithms(was)
    assert (len(public), len(private)) == (3, 1)
    ops._bytes(4)
    assert (len(public), len(private)) == (3, 2)
