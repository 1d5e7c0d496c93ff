"""The bookkeeping of pages on the GPU against a plain loop: everything is equal."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def plain_take(free, table, lengths, counts, page, S):
    """What a take does, on lists: stack, table and lengths change. Gives granted, positions, slots, starts."""
    width, pages = len(table[0]), len(free) - 4
    n_free, needed = max(0, min(free[0], pages)), 0
    granted, starts, positions, slots, taken = [], [0], [], [], 0
    for b, count in enumerate(counts):
        count, length = max(count, 0), max(0, min(lengths[b], width * page))
        had, fits = -(-length // page), length + count <= width * page
        need = -(-(length + count) // page) - had if fits else 0
        needed += need
        ok = fits and (need == 0 or needed <= n_free)
        granted.append(count if ok else 0)
        if ok:
            for k in range(need):
                table[b][had + k] = free[4 + n_free - 1 - (needed - need) - k]
            if need:
                taken = needed
        at = [length + i if i < granted[-1] else -1 for i in range(S)]
        positions.append(at)
        slots.append([table[b][t // page] * page + t % page if t >= 0 and table[b][t // page] >= 0 else -1 for t in at])
        lengths[b] = length + granted[-1]
        starts.append(starts[-1] + granted[-1])
    free[0] = n_free - taken
    return granted, positions, slots, starts


def plain_cut(free, table, lengths, keep, page):
    width, pages = len(table[0]), len(free) - 4
    top = max(0, min(free[0], pages))
    for b in reversed(range(len(lengths))):
        length = max(0, min(lengths[b], width * page))
        lengths[b] = min(length, max(keep[b], 0))
        for at in reversed(range(-(-lengths[b] // page), -(-length // page))):
            if top < pages:
                free[4 + top] = table[b][at]
                top += 1
            table[b][at] = -1
    free[0] = top


class State:
    """A cache, its stack of free pages, and the same as lists."""

    def __init__(self, lengths, page, width, spare, seed=0, bits=8):
        from amdgpu_rustdsl_b200 import Kv4Cache, Kv8Cache
        g = torch.Generator().manual_seed(seed)
        counts = [-(-n // page) for n in lengths]
        used, B = sum(counts), len(lengths)
        order = torch.randperm(used + spare, generator=g).int()
        table = torch.full((B, width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(counts):
            table[b, :n] = order[at:at + n]
            at += n
        free = torch.zeros(4 + max(1, used + spare), dtype=torch.int32)
        free[0], free[4:4 + spare] = spare, order[used:used + spare]
        pool = torch.zeros(max(1, used + spare), 1, (257 if bits == 8 else 136) * page, dtype=torch.uint8, device="cuda")
        self.cache = (Kv8Cache if bits == 8 else Kv4Cache)(pool, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda())
        self.free, self.page = free.cuda(), page
        self.lists = free.tolist(), table.tolist(), list(lengths)

    def same(self):
        free, table, lengths = self.lists
        return self.free.tolist() == free and self.cache.table.tolist() == table and self.cache.lengths.tolist() == lengths

    def take(self, counts, S, positions=torch.int32, **without):
        from amdgpu_rustdsl_b200 import pages_take
        B = self.cache.B
        out = dict(positions=torch.full((B, S), -9, dtype=positions or torch.int32, device="cuda"), slots=torch.full((B, S), -9, dtype=torch.int64, device="cuda"), starts=torch.full((B + 1,), -9, dtype=torch.int32, device="cuda"))
        out = {k: None if k in without or positions is None and k == "positions" else v for k, v in out.items()}
        granted = torch.full((B,), -9, dtype=torch.int32, device="cuda")
        pages_take(self.free, self.cache, torch.tensor(counts, dtype=torch.int32, device="cuda"), granted, **out)
        want = plain_take(*self.lists, counts, self.page, S)
        assert granted.tolist() == want[0]
        for name, x in zip(("positions", "slots", "starts"), want[1:]):
            if out[name] is not None:
                assert out[name].tolist() == x, name
        assert self.same()
        return granted

    def cut(self, keep):
        from amdgpu_rustdsl_b200 import pages_cut
        pages_cut(self.free, self.cache, torch.tensor(keep, dtype=torch.int32, device="cuda"))
        plain_cut(*self.lists, keep, self.page)
        assert self.same()


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("bits", [4, 8])
def test_tokens_come_and_go(page, bits):
    """A few sequences through many steps: single tokens, prompts, drafts that are taken back, ends; pages run out now and then."""
    s = State([0, 5, page, 3 * page + 1, 0], page, 12, 9, bits=bits)
    g = torch.Generator().manual_seed(page)
    for step in range(25):
        most = [1, 4, 3 * page, 1, 0][step % 5]
        counts = torch.randint(0, most + 1, (5,), generator=g).tolist()
        s.take(counts, max(1, most), torch.int64 if step % 2 else torch.int32)
        if step % 3 == 2:
            s.cut([max(0, n - int(torch.randint(0, 5, (1,), generator=g))) for n in s.lists[2]])
        if step % 7 == 6:
            s.cut([0 if b == step % 5 else 1 << 30 for b in range(5)])


@pytest.mark.parametrize("lengths,counts,width,spare", [
    ([0], [1], 1, 0), ([0], [1], 1, 1), ([15], [1], 1, 0), ([16], [1], 1, 5), ([16], [1], 2, 0), ([16, 3, 16], [1, 1, 1], 4, 1), ([16, 3, 16], [1, 1, 1], 4, 2), ([0, 0, 0, 0], [64, 200, 16, 3], 8, 6),
    ([0, 0, 0], [100, 10, 16], 4, 2), ([0, 0], [-5, 0], 4, 2), ([0, 0, 0], [1 << 30, 2147483647, 3], 4, 3)])
def test_pages_run_out_in_order(lengths, counts, width, spare):
    """One that does not fit its table asks for nothing; one that needs more than is left gets none, and so does every one behind it that needs any."""
    s = State(lengths, 16, width, spare)
    s.take(counts, 5)


@pytest.mark.parametrize("B,S,page,L", [(1, 1, 16, 100), (7, 1, 16, 50), (256, 1, 16, 300), (512, 1, 64, 90), (513, 3, 16, 40), (2000, 1, 32, 70), (5000, 2, 16, 33), (3, 5000, 16, 700), (64, 700, 32, 100), (1, 9000, 128, 1)])
def test_batches_of_all_sizes_and_back(B, S, page, L):
    """Then a cut to the lengths before, which leaves everything as it was."""
    g = torch.Generator().manual_seed(B + S)
    lengths, counts = torch.randint(0, L + 1, (B,), generator=g).tolist(), torch.randint(0, S + 1, (B,), generator=g).tolist()
    need = sum(-(-(n + c) // page) + -(n // -page) * -1 for n, c in zip(lengths, counts))
    for spare in {0, need // 2, need, need + 10}:
        s = State(lengths, page, -(-(L + S) // page), max(spare, 1), seed=B)
        s.free[0] = s.lists[0][0] = spare
        before = s.free.clone(), s.cache.table.clone(), s.cache.lengths.clone()
        s.take(counts, S)
        s.cut(lengths)
        assert all(torch.equal(a, b) for a, b in zip(before, (s.free, s.cache.table, s.cache.lengths)))


def test_outputs_that_nobody_asks_for():
    for without in (dict(positions=None), dict(slots=1), dict(starts=1), dict(positions=None, slots=1, starts=1), dict(positions=torch.int64), dict(positions=torch.int64, slots=1)):
        State([20, 3, 0], 16, 8, 9).take([30, 1, 17], 40, **without)


def test_states_that_are_out_of_range_are_cut():
    """Lengths beyond the table or below 0, a height beyond the stack or below 0, entries that name no page: nothing is written outside."""
    s = State([16, 16, 16], 16, 3, 6)
    s.cache.lengths.copy_(torch.tensor([1000, -7, 16], dtype=torch.int32))
    s.lists[2][:] = [1000, -7, 16]
    s.take([1, 1, 1], 2)
    s.free[0] = s.lists[0][0] = 10 ** 6
    s.cache.table[2, 0] = s.lists[1][2][0] = -3
    s.take([0, 20, 3], 4)
    s.free[0] = s.lists[0][0] = 10 ** 6
    s.cut([0, 0, 0])
    s.free[0] = s.lists[0][0] = -5
    s.take([1, 0, 0], 1)
    assert s.lists[0][0] == 0


def test_graphs_and_other_streams():
    """A captured take and cut, replayed; a raw stream."""
    from amdgpu_rustdsl_b200 import pages_cut, pages_take
    s = State([10, 40, 16], 16, 6, 7)
    counts, granted = torch.tensor([9, 9, 1], dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    positions = torch.empty(3, 9, dtype=torch.int32, device="cuda")
    keep = s.cache.lengths.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        pages_take(s.free, s.cache, counts, granted, positions=positions)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        plain_take(*s.lists, [9, 9, 1], 16, 9)
        assert s.same()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    pages_cut(s.free, s.cache, keep, stream=side.cuda_stream)
    side.synchronize()
    plain_cut(*s.lists, [10, 40, 16], 16)   # (three takes handed pages out in turns: they go back in another order)
    assert s.same()


def test_refusals_of_the_python_entry():
    from amdgpu_rustdsl_b200 import pages_cut, pages_take
    s = State([10, 40], 16, 6, 7)
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")
    counts, granted = i32(2), i32(2)
    for call, message in (
            (lambda: pages_take(s.free.long(), s.cache, counts, granted), "int32"), (lambda: pages_take(s.free.cpu(), s.cache, counts, granted), "device"), (lambda: pages_take(s.free[:4], s.cache, counts, granted), "pages"),
            (lambda: pages_take(s.free, s.cache, None, granted), "counts"), (lambda: pages_take(s.free, s.cache, counts, None), "granted"), (lambda: pages_take(s.free, s.cache, i32(3), granted), "counts"),
            (lambda: pages_take(s.free, s.cache, counts, counts), "share memory"), (lambda: pages_take(s.free, s.cache, counts, granted, positions=i32(3, 2)), "positions"), (lambda: pages_take(s.free, s.cache, counts, granted, positions=i32(2, 2).float()), "positions"),
            (lambda: pages_take(s.free, s.cache, counts, granted, slots=i32(2, 2)), "slots"), (lambda: pages_take(s.free, s.cache, counts, granted, positions=i32(2, 3), slots=i32(2, 2).long()), "slots"),
            (lambda: pages_take(s.free, s.cache, counts, granted, positions=i32(2, 0), slots=i32(2, 2).long()), "same S"), (lambda: pages_take(s.free, s.cache, counts, granted, starts=i32(2)), "starts"),
            (lambda: pages_cut(s.free, s.cache, None), "keep"), (lambda: pages_cut(s.free, s.cache, i32(3)), "keep"), (lambda: pages_cut(s.free, s.cache, s.cache.lengths), "share memory")):
        with pytest.raises(ValueError, match=message):
            call()
    assert s.same()
