"""The workspaces that the Python entries keep per stream, with the library and the GPU replaced by stand-ins: no call's kernels come between those of another, and no graph
holds a buffer that may be replaced."""
import ctypes as C
import threading
import time
import types

import pytest
import torch

from amdgpu_rustdsl_b200 import _abi, kv4, ops

CPU = torch.device("cpu")


@pytest.fixture
def no_gpu(monkeypatch):
    """Streams and devices of a machine without a GPU; workspaces are host memory."""
    for module in (ops, kv4):
        monkeypatch.setattr(module, "_raw_stream", lambda torch, dev: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(ops, "_workspace", {})
    monkeypatch.setattr(ops, "_calls", {})


def a_cache():
    cache = object.__new__(kv4.Kv4Cache)
    cache.pool, cache.table, cache.lengths = torch.zeros(4, 1, 136 * 16, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    cache.page, cache.HK, cache.B, cache.capacity, cache.device, cache.c = 16, 1, 1, 64, CPU, _abi.Kv4CacheArgs()
    return cache


class TwoKernels:
    """Calls that write the caller's number to scratch memory, let other threads run, and read it back, as a kernel and the one behind it do in a stream's order."""

    def __init__(self):
        self.wrong = 0

    def call(self, at, number):
        word = C.c_uint32.from_address(at)
        word.value = number
        time.sleep(1e-3)
        self.wrong += word.value != number
        return 0

    def fmha_kv4_attend_workspace(self, cache, a):
        return 64

    def fmha_kv4_attend(self, cache, a, stream, err, cap):
        return self.call(a.workspace, threading.get_ident() & 0xFFFFFFFF)

    def fmha_kv4_evict(self, cache, into, a, stream, err, cap):
        return self.call(a.kept, threading.get_ident() & 0xFFFFFFFF)


def in_threads(work, n=4):
    errors = []

    def run(i):
        try:
            work(i)
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_attention_calls_of_several_threads_do_not_mix(no_gpu, monkeypatch):
    lib = TwoKernels()
    monkeypatch.setattr(_abi, "load", lambda: lib)

    def work(i):
        cache, q = a_cache(), torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16)
        for _ in range(10):
            kv4.fmha_fwd_kv4(q, cache, torch.empty_like(q))
    in_threads(work)
    assert lib.wrong == 0


def test_evictions_of_several_threads_do_not_mix(no_gpu, monkeypatch):
    lib = TwoKernels()
    monkeypatch.setattr(_abi, "load", lambda: lib)

    def work(i):
        cache, weights = a_cache(), torch.zeros(1, 1, 64)
        for _ in range(10):
            kv4.kv4_evict(cache, weights, a_cache(), keep=16)
    in_threads(work)
    assert lib.wrong == 0


def test_splits_of_several_threads_do_not_mix(no_gpu, monkeypatch):
    """The split MXFP8 path launches its two kernels in two calls, at first and when the call is remembered."""
    running, wrong = {}, []

    def launch(kernel, args, grid, stream):
        if kernel == _abi.KVSPLIT:
            running["last"] = threading.get_ident()
            time.sleep(1e-3)
        elif running.get("last") != threading.get_ident():
            wrong.append(kernel)
        return 0
    lib = types.SimpleNamespace(fmha_mxfp8_launch=launch, fmha_mxfp8_validate=lambda *a: 0)
    monkeypatch.setattr(_abi, "load", lambda: lib)

    class Tensor:   # (q has to say that it is on a GPU)
        def __init__(self, x):
            self.x, self.is_cuda = x, True

        def __getattr__(self, name):
            return getattr(self.x, name)

    def work(i):
        q, kv = (Tensor(torch.zeros(1, n, 1, 128, dtype=torch.uint8)) for n in (128, 1024))
        out = Tensor(torch.empty(1, 128, 1, 128, dtype=torch.bfloat16))
        scales = Tensor(torch.zeros(1 << 16, dtype=torch.uint8))
        for _ in range(10):
            assert ops.fmha_fwd_mxfp8(q, kv, kv, scales, scales, scales, out, path="kvsplit", splits=4, check=False) == ("kvsplit", 4)
    in_threads(work)
    assert not wrong


def test_messages_of_several_threads_do_not_mix(no_gpu, monkeypatch):
    def refuse(cache, k, v, S, counts, stream, err, cap):
        C.memmove(err, b"%d rows\0" % S, 8)
        time.sleep(1e-3)
        return 6
    monkeypatch.setattr(_abi, "load", lambda: types.SimpleNamespace(fmha_kv4_append=refuse))

    def work(i):
        cache, x = a_cache(), torch.zeros(1, i + 1, 1, 128, dtype=torch.bfloat16)
        for _ in range(10):
            with pytest.raises(ValueError, match=f"{i + 1} rows"):
                kv4.kv4_append(cache, x, x)
    in_threads(work)


class Captured:
    """A library whose streams are being captured or not, and the scratch memory that its calls were given."""

    def __init__(self):
        self.capturing, self.scratch, self.bytes = False, [], 64

    def cudaStreamIsCapturing(self, stream, status):
        C.cast(status, C.POINTER(C.c_int))[0] = int(self.capturing)
        return 0

    def fmha_kv4_attend_workspace(self, cache, a):
        return self.bytes

    def fmha_kv4_attend(self, cache, a, stream, err, cap):
        self.scratch.append(a.workspace)
        return 0

    def fmha_mxfp8_launch(self, kernel, args, grid, stream):
        if kernel == _abi.KVSPLIT:
            self.scratch.append(args._obj.ptr_ohat)
        return 0


@pytest.fixture
def captured(no_gpu, monkeypatch):
    lib = Captured()
    monkeypatch.setattr(_abi, "load", lambda: lib)
    for module in (ops, kv4):
        monkeypatch.setattr(module, "_raw_stream", lambda torch, dev: 77)   # a stream that is not the default one
    keep = []   # nothing is freed, so that equal addresses are equal buffers

    def empty(*a, **k):
        keep.append(torch.zeros(*a, **k))
        return keep[-1]
    monkeypatch.setattr(torch, "empty", empty)
    return lib


def test_a_captured_attention_call_has_scratch_memory_of_its_own(captured):
    cache, q = a_cache(), torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16)

    def call():
        kv4.fmha_fwd_kv4(q, cache, torch.zeros_like(q))
        return captured.scratch[-1]
    kept = call()
    assert call() == kept
    captured.capturing = True
    first, second = call(), call()
    assert len({kept, first, second}) == 3
    captured.capturing = False
    assert call() == kept       # neither of the graph's buffers stays the stream's
    captured.bytes = 1 << 20
    assert call() not in (kept, first, second)


def test_a_captured_split_is_not_remembered_and_replays_none(captured):
    class Tensor:
        def __init__(self, x):
            self.x, self.is_cuda = x, True

        def __getattr__(self, name):
            return getattr(self.x, name)
    q, kv = (Tensor(torch.zeros(1, n, 1, 128, dtype=torch.uint8)) for n in (128, 1024))
    out, scales = Tensor(torch.zeros(1, 128, 1, 128, dtype=torch.bfloat16)), Tensor(torch.zeros(1 << 16, dtype=torch.uint8))

    def call():
        ops.fmha_fwd_mxfp8(q, kv, kv, scales, scales, scales, out, path="kvsplit", splits=4, check=False)
        return captured.scratch[-1]
    captured.capturing = True
    first = call()
    assert not ops._calls and call() != first
    captured.capturing = False
    kept = call()
    assert kept != first and call() == kept and len(ops._calls) == 1
    captured.capturing = True
    assert call() not in (kept, first)
    captured.capturing = False
    assert call() == kept


def test_buffers_are_made_on_the_stream_that_uses_them(captured, monkeypatch):
    """A buffer for another stream than torch's current one comes from that stream's part of the allocator, which orders its next use."""
    entered = []

    class Stream:
        def __init__(self, handle, device=None):
            self.handle = handle

    class On:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            entered.append(self.stream.handle)

        def __exit__(self, *a):
            entered.append("out")
    monkeypatch.setattr(torch.cuda, "ExternalStream", Stream)
    monkeypatch.setattr(torch.cuda, "stream", On)
    cache, q = a_cache(), torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16)
    kv4.fmha_fwd_kv4(q, cache, torch.zeros_like(q))
    assert entered == []
    kv4.fmha_fwd_kv4(q, cache, torch.zeros_like(q), stream=99)
    assert entered == [99, "out"]
    kv4.fmha_fwd_kv4(q, cache, torch.zeros_like(q), stream=99)
    assert entered == [99, "out"]


def test_workspaces_are_not_dropped_under_a_call(no_gpu, monkeypatch):
    """reset_workspaces from another thread comes behind the call that holds a buffer."""
    lib, events, inside = TwoKernels(), [], threading.Event()

    def attend(cache, a, stream, err, cap):
        inside.set()
        time.sleep(0.05)
        events.append("enqueued")
        return 0
    lib.fmha_kv4_attend = attend
    monkeypatch.setattr(_abi, "load", lambda: lib)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: events.append("dropped"))

    def call():
        q = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16)
        kv4.fmha_fwd_kv4(q, a_cache(), torch.empty_like(q))

    def reset():
        inside.wait(5)
        ops.reset_workspaces()
    in_threads(lambda i: reset() if i else call(), 2)
    assert events == ["enqueued", "dropped"]
