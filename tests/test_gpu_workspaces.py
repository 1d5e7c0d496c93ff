"""The workspaces that the Python entries keep per stream, on the GPU: calls of several threads on one stream, captured graphs beside larger calls."""
import threading

import pytest
import torch

from tests.test_gpu_kv4 import make_cache, no_wait_ran_out, queries  # noqa: F401

pytestmark = pytest.mark.gpu


def in_threads(jobs):
    """Runs the jobs in a thread each, all on the default stream, and hands on what they raise."""
    errors, start = [], threading.Barrier(len(jobs))

    def run(job):
        try:
            start.wait()
            job()
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(job,)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_threads_on_one_stream_get_their_own_results():
    """Attention whose items are cut, decode and prompts, evictions without `kept` and split MXFP8 calls, a few hundred each, against the results of one thread."""
    from amdgpu_rustdsl_b200 import Kv4Cache, fmha_fwd_kv4, fmha_fwd_mxfp8, kv4_evict, kv4_pool
    calls, jobs, checks = 300, [], []

    def attend(seed, S):
        cache, q = make_cache([1500, 700], 2, 64, seed=seed), queries(2, S, 8, seed=seed)
        want, got = torch.empty_like(q), torch.zeros(calls, *q.shape, dtype=torch.bfloat16, device="cuda")
        weights = torch.zeros(2, 2, cache.capacity, device="cuda")
        fmha_fwd_kv4(q, cache, want)
        jobs.append(lambda: [fmha_fwd_kv4(q, cache, out, weights=weights) for out in got])
        checks.append(lambda: (got == want).all())

    def evict(seed):
        cache = make_cache([900, 400], 2, 64, seed=seed)
        weights = torch.rand(2, 2, cache.capacity, generator=torch.Generator().manual_seed(seed)).cuda()

        def into():
            return Kv4Cache(kv4_pool(16, 2), torch.arange(16, device="cuda", dtype=torch.int32).view(2, 8), torch.zeros(2, dtype=torch.int32, device="cuda"))
        want, got = into(), [into() for _ in range(calls)]
        kv4_evict(cache, weights, want, keep=300)
        jobs.append(lambda: [kv4_evict(cache, weights, x, keep=300) for x in got])
        checks.append(lambda: all(torch.equal(x.pool, want.pool) for x in got))

    def split(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        q, k, v = (torch.randint(0, 0x60, (1, n, 4, 128), generator=g, device="cuda").to(torch.uint8) for n in (256, 2048, 2048))
        scales = [torch.cat([torch.full((n * 16,), 120, dtype=torch.uint8, device="cuda"), torch.zeros(640 * 16, dtype=torch.uint8, device="cuda")]) for n in (256, 2048)]
        descale = torch.full((1024,), 0.01, device="cuda")
        want, got = (torch.empty(n, 256, 4, 128, dtype=torch.bfloat16, device="cuda") for n in (1, calls))
        fmha_fwd_mxfp8(q, k, v, *scales, descale, want, path="kvsplit", splits=4)
        jobs.append(lambda: [fmha_fwd_mxfp8(q, k, v, *scales, descale, out[None], path="kvsplit", splits=4) for out in got])
        checks.append(lambda: (got == want).all())

    for seed, S in ((71, 1), (72, 3), (73, 40), (74, 1)):
        attend(seed, S)
    for seed in (75, 76):
        evict(seed)
        split(seed)
    torch.cuda.synchronize()
    in_threads(jobs)
    torch.cuda.synchronize()
    assert all(bool(c()) for c in checks), [bool(c()) for c in checks]


def mxfp8_call(seed):
    """A split MXFP8 call into `out`."""
    from amdgpu_rustdsl_b200 import fmha_fwd_mxfp8
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v = (torch.randint(0, 0x60, (1, n, 4, 128), generator=g, device="cuda").to(torch.uint8) for n in (256, 2048, 2048))
    scales = [torch.cat([torch.full((n * 16,), 120, dtype=torch.uint8, device="cuda"), torch.zeros(640 * 16, dtype=torch.uint8, device="cuda")]) for n in (256, 2048)]
    descale = torch.full((1024,), 0.01, device="cuda")
    out = torch.empty(1, 256, 4, 128, dtype=torch.bfloat16, device="cuda")
    return (lambda **k2: fmha_fwd_mxfp8(q, k, v, *scales, descale, out, path="kvsplit", splits=4, **k2)), out


@pytest.mark.parametrize("warm", [True, False])
def test_a_captured_graph_outlives_larger_calls_on_its_stream(warm):
    """Decode, an eviction without `kept` and a split MXFP8 call are captured, larger calls on the stream replace its workspaces, and tensors take their place: replays leave these alone."""
    from amdgpu_rustdsl_b200 import Kv4Cache, fmha_fwd_kv4, kv4_evict, kv4_pool, reset_workspaces
    reset_workspaces()
    cache, q = make_cache([3000, 1500], 2, 64, seed=81), queries(2, 1, 8)
    weights = torch.rand(2, 2, cache.capacity, generator=torch.Generator().manual_seed(1)).cuda()
    into = [Kv4Cache(kv4_pool(32, 2), torch.arange(32, device="cuda", dtype=torch.int32).view(2, 16), torch.zeros(2, dtype=torch.int32, device="cuda")) for _ in range(2)]
    split, split_out = mxfp8_call(3)
    want, out = torch.empty_like(q), torch.empty_like(q)
    fmha_fwd_kv4(q, cache, want)
    kv4_evict(cache, weights, into[0], keep=1000)
    split()
    split_want = split_out.clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def work():
        fmha_fwd_kv4(q, cache, out)
        kv4_evict(cache, weights, into[1], keep=1000)
        split()
        split(fused_combine=True)
    with torch.cuda.stream(side):
        if warm:
            work()
            work()   # (the split calls are remembered)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        work()
    with torch.cuda.stream(side):
        big_cache, big = make_cache([2000] * 4, 2, 64, seed=82), queries(4, 300, 16)
        big_out = torch.empty_like(big)
        fmha_fwd_kv4(big, big_cache, big_out, weights=torch.zeros(4, 2, big_cache.capacity, device="cuda"))
        kv4_evict(big_cache, torch.rand(4, 2, big_cache.capacity, device="cuda"), Kv4Cache(kv4_pool(128, 2), torch.arange(128, device="cuda", dtype=torch.int32).view(4, 32),
                                                                                         torch.zeros(4, dtype=torch.int32, device="cuda")), keep=2000)
        reset_workspaces()
        marks = [torch.full((n << 10,), 0xA5, dtype=torch.uint8, device="cuda") for n in (1, 16, 64, 256, 1024, 2048, 4096, 8192, 16384) for _ in range(8)]
    torch.cuda.synchronize()
    for _ in range(3):
        out.zero_(), split_out.zero_(), into[1].pool.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(split_out, split_want) and torch.equal(into[1].pool, into[0].pool)
    assert all(bool((m == 0xA5).all()) for m in marks)


def test_graphs_captured_from_one_stream_run_side_by_side():
    """Two graphs that torch captures from the same stream, replayed on two streams at the same time: neither writes to the other's workspace."""
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    graphs = []
    for seed in (91, 92):
        cache, q = make_cache([4000, 3000], 2, 64, seed=seed), queries(2, 1, 8, seed=seed)
        want, out = torch.empty_like(q), torch.empty_like(q)
        fmha_fwd_kv4(q, cache, want)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):   # (torch's own stream for captures)
            for _ in range(20):
                fmha_fwd_kv4(q, cache, out)
        graphs.append((graph, torch.cuda.Stream(), want, out, cache, q))
    for _ in range(20):
        for graph, stream, _, _, _, _ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, _, want, out, _, _ in graphs)


def test_a_stream_that_is_not_the_current_one():
    """`stream=`: the workspace grows while the stream is still at work, and other tensors of the current stream come and go."""
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    cache = make_cache([3000, 1500], 2, 64, seed=83)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for S in (1, 5, 40, 300):
        q = queries(2, S, 8)
        want = torch.empty_like(q)
        fmha_fwd_kv4(q, cache, want)
        outs = torch.zeros(20, *q.shape, dtype=torch.bfloat16, device="cuda")
        torch.cuda.synchronize()
        for out in outs:
            fmha_fwd_kv4(q, cache, out, stream=side.cuda_stream)
            torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        assert (outs == want).all()
