"""The operators around the 8-bit cache at the edges of how their work is shared, used from several threads, streams and graphs, and together as a server uses them (references and tolerances:
test_gpu_kv8.py)."""
import pytest
import torch

from tests import test_gpu_kv8 as K
from tests.test_gpu_kv8 import no_wait_ran_out  # noqa: F401
from tests.test_gpu_workspaces import in_threads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,HK,H,L,S", [(1, 1, 4, 20011, 40), (1, 2, 6, 9001, 333), (1, 4, 12, 4001, 170), (1, 8, 24, 2001, 333), (1, 1, 3, 30001, 85), (1, 1, 16, 12000, 2), (2, 1, 1, 6000, 33)])
def test_items_of_many_parts(B, HK, H, L, S):
    """Few items, each of which many CTAs have a part of: up to 148 of 40 rows, 18, 9 and 4 of 256."""
    K.test_many_tiles_against_a_plain_product(B, HK, H, L, S)


@pytest.mark.parametrize("width", [4, 5])
@pytest.mark.parametrize("S,group", [(1, 4), (1, 16), (2, 16), (8, 4), (3, 7)])
def test_items_at_the_length_from_which_they_are_cut(width, S, group):
    """Tables of 512 tokens, whose items stay whole, and of 640, whose items are cut."""
    cache = K.make_cache([512, 511, 0, 1, 385, 128, 129, 16], 2, 128, seed=50, width=width)
    K.check_attend(cache, K.queries(8, S, 2 * group))
    K.check_attend(cache, K.queries(8, S, 2 * group), counts=[S, 0, 1, 1, S - 1, -1, 100, S])


@pytest.mark.parametrize("S,group,HK", [(1, 2, 1), (5, 1, 2), (9, 4, 1)])
def test_thousands_of_short_sequences(S, group, HK):
    """More items than CTAs by far, many of them empty."""
    g = torch.Generator().manual_seed(51)
    lengths = torch.randint(0, 40, (1500,), generator=g)
    lengths[torch.rand(1500, generator=g) < 0.3] = 0
    lengths[7] = 150
    cache = K.make_cache(lengths.tolist(), HK, 16, seed=52)
    K.check_attend(cache, K.queries(1500, S, HK * group))


def test_a_batch_of_empty_sequences():
    from amdgpu_rustdsl_b200 import fmha_fwd_kv8, kv8_append, kv8_read
    cache = K.make_cache([64, 64, 64], 2, 32, seed=53)
    cache.lengths.zero_()
    before = cache.pool.clone()
    for S in (1, 40):
        q, k = K.queries(3, S, 8), torch.ones(3, S, 2, 128, dtype=torch.bfloat16, device="cuda")
        out, lse = torch.full_like(q, float("nan")), torch.zeros(3, 8, S, device="cuda")
        kv8_append(cache, k, k)
        fmha_fwd_kv8(q, cache, out, lse=lse)
        kv8_read(cache, k, k, last=True)
        assert (out == 0).all() and (lse == -float("inf")).all() and (k == 0).all()
    assert torch.equal(cache.pool, before)


def test_no_rows_at_all():
    """S of 0: every call is a call that does nothing."""
    from amdgpu_rustdsl_b200 import fmha_fwd_kv8, kv8_append, kv8_read
    cache = K.make_cache([20, 3], 2, 16, seed=54)
    before, none = cache.pool.clone(), torch.empty(2, 0, 2, 128, dtype=torch.bfloat16, device="cuda")
    kv8_append(cache, none, none)
    kv8_read(cache, none, none)
    q = torch.empty(2, 0, 8, 128, dtype=torch.bfloat16, device="cuda")
    fmha_fwd_kv8(q, cache, torch.empty_like(q), lse=torch.empty(2, 8, 0, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(cache.pool, before)


def test_appends_of_more_than_there_is():
    """counts beyond the rows and below 0: cut to the rows, the length, and 0."""
    g = torch.Generator().manual_seed(55)
    cache = K.make_cache([30, 2, 17, 64], 2, 16, seed=55)
    k, v = (torch.randn(4, 5, 2, 128, generator=g).bfloat16().cuda() for _ in range(2))
    K.check_append(cache, k, v, counts=[100, 4, -7, 0x7FFFFFFF])


def test_threads_on_one_stream_get_their_own_results():
    """Decode and prompts whose items are cut, appends and rotations, a few hundred each from a thread of its own, against the results of one thread."""
    from amdgpu_rustdsl_b200 import Rope, fmha_fwd_kv8, kv8_append, rope_rotate
    calls, jobs, checks = 200, [], []

    def attend(seed, S):
        cache, q = K.make_cache([1500, 700], 2, 64, seed=seed), K.queries(2, S, 8, seed=seed)
        want, got = torch.empty_like(q), torch.zeros(calls, *q.shape, dtype=torch.bfloat16, device="cuda")
        fmha_fwd_kv8(q, cache, want)
        jobs.append(lambda: [fmha_fwd_kv8(q, cache, out) for out in got])
        checks.append(lambda: (got == want).all())

    def append(seed):
        cache, other = (K.make_cache([500, 100], 2, 64, seed=seed) for _ in range(2))
        k = K.queries(2, 30, 2, seed=seed)
        kv8_append(other, k, k)
        jobs.append(lambda: [kv8_append(cache, k, k) for _ in range(calls)])
        checks.append(lambda: torch.equal(cache.pool, other.pool))

    def rotate(seed):
        rope, x, at = Rope(128), K.queries(2, 30, 4, seed=seed), torch.arange(60, device="cuda").view(2, 30)
        want, got = rope_rotate(rope, x, at, torch.empty_like(x)), torch.zeros(calls, *x.shape, dtype=torch.bfloat16, device="cuda")
        jobs.append(lambda: [rope_rotate(rope, x, at, out) for out in got])
        checks.append(lambda: (got == want).all())

    for seed, S in ((61, 1), (62, 6), (63, 40), (64, 300)):
        attend(seed, S)
    append(65)
    rotate(66)
    torch.cuda.synchronize()
    in_threads(jobs)
    torch.cuda.synchronize()
    assert all(bool(c()) for c in checks), [bool(c()) for c in checks]


def test_streams_at_once():
    """Calls of two streams that overlap, decode and prompts: each stream has its own workspace."""
    from amdgpu_rustdsl_b200 import fmha_fwd_kv8
    work = []
    for seed, S in ((67, 1), (68, 200), (69, 4), (70, 48)):
        cache, q = K.make_cache([2500, 900], 2, 64, seed=seed), K.queries(2, S, 8, seed=seed)
        want = torch.empty_like(q)
        fmha_fwd_kv8(q, cache, want)
        work.append((cache, q, want, [torch.zeros_like(q) for _ in range(50)]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(50):
        for x, (cache, q, _, outs) in enumerate(work):
            with torch.cuda.stream(streams[(x + i) % 2]):
                fmha_fwd_kv8(q, cache, outs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, _, want, outs in work for out in outs)


def test_a_step_takes_no_memory_once_it_has_run():
    from amdgpu_rustdsl_b200 import Rope, fmha_fwd_kv8, kv8_append, pages_cut, pages_stack, pages_take, rope_rotate
    cache, rope = K.make_cache([900, 300], 2, 64, seed=71, width=20), Rope(128)
    free, keep, granted = pages_stack(9), cache.lengths.clone(), torch.zeros_like(cache.lengths)
    steps = []
    for S in (1, 48):
        q, k = K.queries(2, S, 8), K.queries(2, S, 2)
        steps.append((q, k, torch.empty_like(q), torch.full_like(granted, S), torch.empty(2, S, dtype=torch.int32, device="cuda")))

    def run():
        for q, k, out, counts, positions in steps:
            pages_take(free, cache, counts, granted, positions=positions)
            rope_rotate(rope, q, positions, y=k)
            kv8_append(cache, k, k, counts=granted)
            fmha_fwd_kv8(q, cache, out, counts=granted)
            pages_cut(free, cache, keep)
    run()
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    for _ in range(3):
        run()
    torch.cuda.synchronize()
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before


def test_decode_steps_of_a_captured_graph():
    """pages_take, rope_rotate, kv8_append and fmha_fwd_kv8 captured once and replayed for 70 tokens, page ends among them, beside the same steps launched one by one; graphs of two batches that
    replay in turn do not disturb one another. Sequences stop at different times, and one runs out of its table."""
    from amdgpu_rustdsl_b200 import Rope
    from amdgpu_rustdsl_b200.kv8_example import PagedBatch
    B, HK, H = 5, 2, 8
    rope = Rope(128, scaling={"kind": "linear", "factor": 2.0})

    def batch():
        x = PagedBatch(B, 2, HK, 60, 90, rope, page=16)
        start, rows = torch.tensor([1, 16, 30, 0, 64], dtype=torch.int32, device="cuda"), 64
        x.begin(start, rows)
        g = torch.Generator(device="cuda").manual_seed(72)
        for i in range(2):
            q = torch.randn(B, rows, H, 128, generator=g, device="cuda").bfloat16()
            k, v = (torch.randn(B, rows, HK, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
            x.layer(i, q, k, v, torch.empty_like(q))
        return x

    def step(x, q, k, v, counts, outs):
        x.begin(counts, 1)
        for i in range(2):
            x.layer(i, q[i].clone(), k[i].clone(), v[i], outs[i])

    eager, captured = batch(), [batch(), batch()]
    inputs = [[torch.zeros(2, B, 1, h, 128, dtype=torch.bfloat16, device="cuda") for h in (H, HK, HK)] + [torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(2, B, 1, H, 128, dtype=torch.bfloat16, device="cuda")] for _ in range(3)]
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in captured]
    for x, data, graph in zip(captured, inputs, graphs):
        with torch.cuda.graph(graph):
            step(x, *data)
    g = torch.Generator(device="cuda").manual_seed(73)
    for t in range(70):
        new = [torch.randn(2, B, 1, h, 128, generator=g, device="cuda").bfloat16() for h in (H, HK, HK)]
        counts = torch.tensor([1, 1, t % 2, int(t < 20), 1], dtype=torch.int32, device="cuda")
        for data in inputs:
            for x, y in zip(data, new + [counts]):
                x.copy_(y)
        step(eager, *inputs[2])
        for graph in graphs:
            graph.replay()
        for x, data in zip(captured, inputs):
            assert torch.equal(x.lengths, eager.lengths) and torch.equal(x.granted, eager.granted) and torch.equal(x.free, eager.free) and torch.equal(x.table, eager.table)
            assert torch.equal(data[4], inputs[2][4]), t
    assert eager.lengths.tolist() == [71, 86, 65, 20, 96]
    assert all(torch.equal(a.pool, b.pool) for x in captured for a, b in zip(x.caches, eager.caches))
