"""The workspaces that the Python entries keep per stream, on the GPU: calls of several threads on one stream."""
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
