"""Scratch memory that the package lends to its calls, without a GPU: the entry points run against stand-ins for the
library's functions and for torch's streams, which record who enqueues when on what buffer."""
import contextlib
import ctypes as C
import importlib
import threading

import pytest
import torch

import gemmkernels_b200 as GK
from gemmkernels_b200 import _lib as L
from gemmkernels_b200 import Layout, Operator

# (the package's `matmul` is the function, not the module)
matmul_mod, fused_mod, contract_mod = (importlib.import_module(f"gemmkernels_b200.{m}") for m in ("matmul", "fused", "contract"))
F16, F32 = GK.Float16, GK.Float32


class FakeStream:
    def __init__(self, cuda_stream=0):
        self.cuda_stream = cuda_stream


@pytest.fixture
def no_gpu(monkeypatch):
    """torch's streams and devices as far as the entry points use them; buffers are host tensors."""
    monkeypatch.setattr(torch.cuda, "device", lambda *a: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "stream", lambda *a: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda s, device=None: FakeStream(s))
    monkeypatch.setattr(torch.cuda, "default_stream", lambda *a: FakeStream())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: FakeStream())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    for mod in (matmul_mod, fused_mod, contract_mod):
        monkeypatch.setattr(mod, "handle", lambda *a: C.c_void_p(1))
    monkeypatch.setattr(matmul_mod, "_workspaces", {})


class Recorder:
    """A library function that enqueues twice, as the calls with scratch do (its contents, then the product), and
    gives another thread the time to come in between."""

    def __init__(self):
        self.log, self.met = [], threading.Barrier(2)

    def __call__(self, ws):
        me = threading.get_ident()
        self.log.append((me, ws))
        with contextlib.suppress(threading.BrokenBarrierError):
            self.met.wait(timeout=0.3)
        self.log.append((me, ws))
        return L.GK_OK


def two_threads(*calls):
    errors = []

    def guarded(f):
        try:
            f()
        except Exception as e:      # noqa: BLE001 - reported by the assertion below
            errors.append(e)

    threads = [threading.Thread(target=guarded, args=(f,)) for f in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def cm(*shape, dtype=torch.float16):
    return torch.zeros(tuple(reversed(shape)), dtype=dtype).permute(*reversed(range(len(shape))))


class FakeCall:
    device = torch.device("cpu")

    def __init__(self, recorder):
        self.function = lambda ws, n, s: recorder(ws)

    def workspace_bytes(self, h):
        return 64

    def arguments(self, h, ws, n):
        return ws, n


def entry_point(which, rec, monkeypatch):
    """A callable (stream) -> None that goes through the entry point with `rec` as the library's function."""
    def query(*args):
        args[-1]._obj.workspace_bytes = 4096
        return L.GK_OK

    if which == "layer":
        return lambda s: fused_mod._run(FakeCall(rec), s)
    if which == "product":
        monkeypatch.setattr(L.lib, "gk_gemm_query", query)
        monkeypatch.setattr(L.lib, "gk_gemm", lambda h, desc, a, b, c, d, epi, ws, n, s: rec(ws))
        cf = GK.get_config(gemm_shape=(64, 64, 4096), operator=Operator.TCGen05Operator[F16, F32], global_a_layout=Layout.ColMajor[F16],
                           global_b_layout=Layout.ColMajor[F16], global_c_layout=Layout.Zero[F32], global_d_layout=Layout.ColMajor[F32])
        return lambda s: GK.matmul(cf, cm(64, 4096), cm(4096, 64), None, cm(64, 64, dtype=torch.float32), stream=s)
    monkeypatch.setattr(L.lib, "gk_contract_query", query)
    monkeypatch.setattr(L.lib, "gk_contract", lambda h, desc, a, b, c, d, ws, n, s: rec(ws))
    return lambda s: GK.contract_(cm(8, 8, dtype=torch.float32), "ab", cm(8, 8), "ac", cm(8, 8), "cb", stream=s)


@pytest.mark.parametrize("which", ["layer", "product", "contraction"])
def test_calls_of_two_threads_on_one_stream_do_not_mix(which, no_gpu, monkeypatch):
    """Both write their scratch and read it in a later launch: the pairs must not interleave."""
    rec = Recorder()
    call = entry_point(which, rec, monkeypatch)
    two_threads(lambda: call(5), lambda: call(5))
    (a, wa), (b, wb), (c, wc), (d, wd) = rec.log
    assert a == b and c == d and a != c
    assert wa == wb == wc == wd and wa      # the same buffer: never one per call


@pytest.mark.parametrize("which", ["layer", "product", "contraction"])
def test_streams_have_buffers_of_their_own_and_do_not_wait(which, no_gpu, monkeypatch):
    rec = Recorder()
    call = entry_point(which, rec, monkeypatch)
    two_threads(lambda: call(5), lambda: call(6))
    assert len(rec.log) == 4 and len({t for t, _ in rec.log[:2]}) == 2 and len({w for _, w in rec.log}) == 2


def test_a_call_that_fails_gives_the_buffer_back(no_gpu):
    def fails(*_):
        raise RuntimeError("refused")

    call = FakeCall(Recorder())
    call.function = fails
    for _ in range(2):
        with pytest.raises(RuntimeError, match="refused"):
            fused_mod._run(call, 5)


@pytest.mark.parametrize("which", ["layer", "product", "contraction"])
def test_captured_calls_have_scratch_of_their_own(which, no_gpu, monkeypatch):
    """A buffer that two graphs share would be written by both when they are replayed at the same time, and one that a graph's
    memory pool holds must not be lent to calls outside the graph."""
    capturing, seen, kept = [False], [], []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    real_empty = torch.empty

    def empty(*size, **kw):
        t = real_empty(*size, **kw)
        if kw.get("dtype") == torch.uint8:
            kept.append(t)                   # alive, so that no two buffers can have one address
        return t

    monkeypatch.setattr(torch, "empty", empty)
    call = entry_point(which, lambda ws: seen.append(ws) or L.GK_OK, monkeypatch)
    for state in (False, True, True, False):
        capturing[0] = state
        call(5)
    eager, first, second, again = seen
    assert eager == again and len({eager, first, second}) == 3 and all(seen)
    capturing[0] = True
    call(7)                                  # the first call on a stream is a captured one
    capturing[0] = False
    call(7)
    assert seen[-1] != seen[-2]


@pytest.mark.parametrize("off_a,off_b", [(0, 0), (2, 0), (0, 14), (8, 6)])
@pytest.mark.parametrize("bound", [False, True])
def test_room_for_the_copies_of_operands_off_16_bytes(off_a, off_b, bound, no_gpu, monkeypatch):
    """Aligned leading dimensions, a base between two 16-byte boundaries: the call asks for such a product, and gets the room."""
    asked, got = [], []

    def query(h, desc, fused, groups, plan):
        d = desc._obj
        asked.append((d.lda % 8 != 0, d.ldb % 8 != 0))
        plan._obj.workspace_bytes = 512 * (d.lda % 8 != 0) + 1024 * (d.ldb % 8 != 0)
        return L.GK_OK

    monkeypatch.setattr(L.lib, "gk_gemm_fused_query", query)
    desc = L.GemmDesc(m=64, n=64, k=64, lda=64, ldb=64, ldd=64, alpha=1.0)
    call = fused_mod._Call(desc, L.FusedDesc(), None, (0x1000 + off_a, 0x2000 + off_b, None, 0x3000), torch.device("cpu"), ())
    call.function = lambda h, desc, fu, gr, a, b, c, d, ws, n, s: got.append(getattr(n, "value", n)) or L.GK_OK
    if bound:
        fused_mod.BoundFused(call)(5)
    else:
        fused_mod._run(call, 5)
    want = 512 * (off_a != 0) + 1024 * (off_b != 0)
    assert got == [want] and (not want or asked == [(off_a != 0, off_b != 0)])
    assert (desc.lda, desc.ldb) == (64, 64)


@pytest.mark.parametrize("which", ["layer", "product", "contraction"])
def test_bound_calls_use_scratch_of_the_stream_they_are_on(which, no_gpu, monkeypatch):
    """A buffer allocated under one stream and used on another may still be in use there, and goes back to the first
    when the object is dropped: each buffer must be allocated under the stream that it is used on, once."""
    on, made, used, capturing = [0], [], [], [False]

    @contextlib.contextmanager
    def stream(s):
        before, on[0] = on[0], s.cuda_stream
        yield
        on[0] = before

    real_empty = torch.empty

    def empty(*size, **kw):
        t = real_empty(*size, **kw)
        if kw.get("dtype") in (torch.uint8, torch.int64):
            made.append((t.data_ptr(), on[0], t))
        return t

    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(torch, "empty", empty)
    address = lambda ws: ws if isinstance(ws, int) else ws.value
    rec = lambda ws: used.append(address(ws)) or L.GK_OK
    entry_point(which, rec, monkeypatch)
    if which == "layer":
        call = FakeCall(rec)
        call.arguments = lambda h, ws, n: (ws, n)
        bound = fused_mod.BoundFused(call)
    elif which == "product":
        cf = GK.get_config(gemm_shape=(64, 64, 4096), operator=Operator.TCGen05Operator[F16, F32], global_a_layout=Layout.ColMajor[F16],
                           global_b_layout=Layout.ColMajor[F16], global_c_layout=Layout.Zero[F32], global_d_layout=Layout.ColMajor[F32])
        bound = GK.bind(cf, cm(64, 4096), cm(4096, 64), None, cm(64, 64, dtype=torch.float32))
    else:
        bound = GK.bind_contract(cm(8, 8, dtype=torch.float32), "ab", cm(8, 8), "ac", cm(8, 8), "cb")
    for s in (0, 5, 6, 5, 0):
        bound(s)
    owner = {p: s for p, s, _ in made}
    assert [owner[p] for p in used] == [0, 5, 6, 5, 0] and len(made) == 3
    capturing[0] = True
    bound(5)
    capturing[0] = False
    assert used[-1] == made[-1][0] and len(made) == 4      # a graph's own
    bound(5)
    assert used[-1] == used[1] and len(made) == 4


def test_plans_are_made_on_the_device_of_the_arrays(no_gpu, monkeypatch):
    """Planning raises the shared-memory limits of the kernels it chooses, on the device that is current, and remembers that
    it did in the handle of the arrays' device: on another one the later launch would fail."""
    current, planned = [0], []

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], getattr(d, "index", d)
        yield
        current[0] = before

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(L.lib, "gk_gemm_fused_query", lambda *a: planned.append(current[0]) or L.GK_OK)
    monkeypatch.setattr(fused_mod, "_one_device", lambda *a: torch.device("cuda", 1))
    cf = GK.get_config(gemm_shape=(64, 40, 32), operator=Operator.TCGen05Operator[F16, F32], global_a_layout=Layout.ColMajor[F16],
                       global_b_layout=Layout.ColMajor[F16], global_c_layout=Layout.Zero[F32], global_d_layout=Layout.ColMajor[F32])
    GK.query(cf, cm(64, 32), cm(32, 40), None, cm(64, 40, dtype=torch.float32), epilogue=GK.Epilogue.BiasActivationResidual())
    GK.grouped_query(cf, cm(64, 32, 2), cm(32, 40), None, cm(64, 40, dtype=torch.float32), torch.zeros(3, dtype=torch.int32))
    assert planned == [1, 1] and current[0] == 0
