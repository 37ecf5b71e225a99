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


def test_calls_that_would_be_read_out_of_range_are_refused(host):
    """Tensors that hold less than the call says, lie in other strides than it can say, or on another device."""
    class Elsewhere(torch.Tensor):
        get_device = lambda self: 1
    away = lambda t: t.clone().as_subclass(Elsewhere)
    N, K, M = 200, 256, 40
    q, s = torch.zeros(N, K, dtype=torch.uint8), torch.ones(2, 2)
    W = ops.GMat(ops.FMT_FP8_B128, N, K, q, s)
    xq, xs = torch.zeros(M, K, dtype=torch.uint8), torch.ones(2, M)
    ws, y = torch.zeros(4096, dtype=torch.uint8), torch.zeros(M, N)
    ok = [lambda: ops.fp8_gemm(W, xq, xs, y=y, ws=ws), lambda: ops.fp8_gemm(W, xq, torch.ones(2, M + 3)[:, :M]), lambda: ops.fp8_gemm(W, xq[:1], torch.ones(2, M))]
    refused(*(lambda a=a: ops.GMat(ops.FMT_FP8_B128, N, K, *a) for a in ((q[:199], s), (q, s[:1]), (q, s.double()), (q.short(), s), (q.t().contiguous().t(), s), (q, s.t().contiguous().t()))),
            lambda: ops.fp8_gemm(W, xq, torch.ones(2, M + 3)[:, :M - 1]), lambda: ops.fp8_gemm(W, xq, torch.ones(1, M - 1)), lambda: ops.fp8_gemm(W, xq, xs, ws=ws[:4095]),
            lambda: ops.fp8_gemm(W, xq, xs, ws=torch.zeros(8192, dtype=torch.uint8)[::2]), lambda: ops.fp8_gemm(W, xq, away(xs)), lambda: ops.fp8_gemm(W, xq, xs, y=away(y)),
            lambda: ops.fp8_gemm(W, xq, xs, ws=away(ws)), lambda: ops.fp8_gemm(ops.GMat(ops.FMT_FP8_B128, N, K, away(q), s), xq, xs),
            lambda: ops.fp8_gemm(ops.GMat(ops.FMT_FP8_B128, N, K, q, away(s)), xq, xs), lambda: ops.fp8_gemm(W, away(xq), xs))
    bf = torch.zeros(M, K, dtype=torch.bfloat16)
    ok += [lambda: ops.fp8_quant_rows(bf, q=xq, s=xs), lambda: ops.fp8_quantize(bf)]
    refused(lambda: ops.fp8_quant_rows(bf, q=away(xq)), lambda: ops.fp8_quant_rows(bf, s=away(xs)), lambda: ops.fp8_quantize(bf, q=away(xq)), lambda: ops.fp8_quantize(bf, s=away(torch.ones(1, 2))))
    lgt, bias = torch.zeros(M, 64), torch.zeros(64)
    i, w = torch.zeros(M, 2, dtype=torch.int32), torch.zeros(M, 2)
    ok += [lambda: ops.router_grouped_topk(lgt, 2, bias=bias, ids=i, w=w)]
    refused(lambda: ops.router_grouped_topk(lgt, 2, bias=away(bias)), lambda: ops.router_grouped_topk(lgt, 2, ids=away(i)), lambda: ops.router_grouped_topk(lgt, 2, w=away(w)),
            lambda: ops.router_grouped_topk(lgt, 2, score="tanh"))
    tab = torch.zeros(6, dtype=torch.int64)
    out = torch.zeros(M, K, dtype=torch.bfloat16)
    moe = lambda **k: ops.moe_fp8(**{**dict(ids=i, w=w, rec_tab=tab, li=1, E=3, x=bf, H=K, I=128, shared=bf), **k})
    ok += [moe, lambda: moe(lg=torch.zeros(M)), lambda: moe(lg=torch.zeros(M, 5), col=4), lambda: moe(lg=torch.zeros(M, 9)[:, 2:5], col=2), lambda: moe(lg=torch.zeros(M, 5)[:, 1]),
           lambda: moe(ws=ws, out=out), lambda: moe(lg=torch.zeros(M, 5)[:, 1:2])]
    refused(lambda: moe(lg=torch.zeros(5, M).t(), col=2), lambda: moe(lg=torch.zeros(M, 10)[:, ::2], col=1), lambda: moe(lg=torch.zeros(M, 9)[:, :3], col=3), lambda: moe(lg=torch.zeros(M), col=1),
            lambda: moe(rec_tab=torch.zeros(12, dtype=torch.int64)[::2]), lambda: moe(ws=ws[1:]), *(lambda k=k, v=v: moe(**{k: away(v)}) for k, v in
            dict(ids=i, w=w, rec_tab=tab, shared=bf, lg=torch.zeros(M), out=out, ws=ws, x=bf).items()))
    for c in ok:
        with pytest.raises(Seen):
            c()


def test_a_record_is_bytes_in_one_piece(host):
    u8, s = torch.zeros(256, 256, dtype=torch.uint8), torch.ones(2, 2)
    n = ops.Fp8RecLayout(256, 256).total
    make = lambda out: ops.fp8_record(256, 256, (u8, s), (u8, s), (u8, s), out=out)
    room = torch.full((n + 32,), 7, dtype=torch.uint8)
    assert make(room[16:]).data_ptr() == room.data_ptr() + 16 and (room[:16] == 7).all() and (room[n + 16:] == 7).all()
    refused(lambda: make(torch.zeros(n - 1, dtype=torch.uint8)), lambda: make(torch.zeros(n)), lambda: make(torch.zeros(2 * n, dtype=torch.uint8)[::2]), lambda: make(torch.zeros(1, n, dtype=torch.uint8)))
