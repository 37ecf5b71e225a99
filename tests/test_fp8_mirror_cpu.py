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


class Seen(Exception):
    """A call that has come as far as the library."""


@pytest.fixture
def host(monkeypatch):
    """The mirror on CPU tensors: their device takes the place of the current one, and the library only counts what reaches it."""
    class Lib:
        def __getattr__(self, name):
            if name.endswith("_ws_bytes"):
                return lambda *a: 4096

            def call(*a):
                raise Seen(name)
            return call

    class Ctx:
        device, handle = -1, None

        def check(self, st):
            raise AssertionError("not reached")
    from eke_hive_b200 import _lib
    real = _lib.load()
    fake = Lib()
    fake.hb_fp8_rec_layout_make = real.hb_fp8_rec_layout_make
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(ops, "_raw_stream", lambda d: 0)
    monkeypatch.setattr(ops, "_CTX", {-1: Ctx()})
    monkeypatch.setattr(ops, "_lib_handle", fake)
    monkeypatch.setattr(ops, "_empty_strided", lambda size, stride, dtype: torch.empty_strided(size, stride, dtype=dtype))
    monkeypatch.setattr(ops, "_p", lambda t: None if t is None else t.data_ptr())


def refused(*calls):
    for c in calls:
        with pytest.raises(ops.HbError):
            c()


def test_wrong_types_are_errors_of_the_library(host):
    bf, u8 = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(256, 256, dtype=torch.uint8)
    for ok in (lambda: ops.fp8_quant_rows(bf), lambda: ops.fp8_quantize(bf), lambda: ops.fp8_quantize(bf.float())):
        with pytest.raises(Seen):
            ok()
    refused(lambda: ops.fp8_quant_rows(bf.float()), lambda: ops.fp8_quantize(bf.half()), lambda: ops.fp8_quantize(bf[:, :128]))
    s = torch.ones(2, 2)
    assert ops.fp8_record(256, 256, (u8, s), (u8, s), (u8, s)).numel() == ops.Fp8RecLayout(256, 256).total
    for bad in ((u8[:128], s), (u8.float(), s), (u8, s[:1]), (u8, s.double())):
        refused(lambda: ops.fp8_record(256, 256, bad, (u8, s), (u8, s)), lambda: ops.fp8_record(256, 256, (u8, s), (u8, s), bad))
    ids, w, tab = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(Seen):
        ops.moe_fp8(ids, w, tab, 0, 3, bf, 256, 128, shared=bf)
    refused(lambda: ops.moe_fp8(ids, w, tab, 0, 3, bf, 256, 128, shared=bf, out_dtype=torch.float32))
