"""Cuts of tables with entries that name no page: what goes back onto the stack is pages, each once, and what is handed out later is pages. (The loop is test_gpu_pages.py's but for such entries.)"""
import pytest
import torch

from tests import test_gpu_pages as P

pytestmark = pytest.mark.gpu


def plain_cut(free, table, lengths, keep, page, pool):
    width, pages = len(table[0]), len(free) - 4
    top = max(0, min(free[0], pages))
    for b in reversed(range(len(lengths))):
        length = max(0, min(lengths[b], width * page))
        lengths[b] = min(length, max(keep[b], 0))
        for at in reversed(range(-(-lengths[b] // page), -(-length // page))):
            if 0 <= table[b][at] < pool and top < pages:
                free[4 + top] = table[b][at]
                top += 1
            table[b][at] = -1
    free[0] = top


@pytest.mark.parametrize("B,page,L,part", [(1, 16, 100, 0.5), (1, 16, 20000, 0.3), (3, 16, 9000, 0.2), (5, 32, 400, 1.0), (15, 16, 3000, 0.5), (16, 16, 2500, 0.1), (17, 16, 700, 0.5), (70, 64, 900, 0.5),
                                           (512, 16, 60, 0.5), (513, 16, 40, 0.5), (1025, 128, 700, 0.1), (2000, 16, 33, 0.5), (4, 128, 130, 0.0)])
@pytest.mark.parametrize("keeps", ["nothing", "some", "one page less"])
def test_entries_that_name_no_page(B, page, L, part, keeps):
    from amdgpu_rustdsl_b200 import pages_cut
    g = torch.Generator().manual_seed(B + L)
    lengths = torch.randint(0, L + 1, (B,), generator=g).tolist()
    s = P.State(lengths, page, -(-L // page), 5, seed=B)
    pool = s.cache.pool.shape[0]
    table = s.cache.table.cpu()
    lost = torch.rand(table.shape, generator=g) < part
    table[lost] = torch.tensor([-1, -2 ** 31, 2 ** 31 - 1, pool], dtype=torch.int32)[torch.randint(0, 4, (int(lost.sum()),), generator=g)]
    s.cache.table.copy_(table)
    s.lists[1][:] = table.tolist()
    keep = [0 if keeps == "nothing" else max(0, n - page) if keeps == "one page less" else int(torch.randint(0, n + 1, (1,), generator=g)) for n in lengths]
    pages_cut(s.free, s.cache, torch.tensor(keep, dtype=torch.int32, device="cuda"))
    plain_cut(*s.lists, keep, page, pool)
    assert s.same()
    height = s.lists[0][0]
    stack = s.lists[0][4:4 + height]
    assert len(set(stack)) == height and all(0 <= x < pool for x in stack)


def test_a_length_without_pages_harms_nobody_else():
    """A length that was raised by hand past the pages of its sequence: after a cut and a take, every granted token has a page."""
    from amdgpu_rustdsl_b200 import pages_cut, pages_take
    s = P.State([16, 16], 16, 8, 1)
    s.cache.lengths[0] = 100
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    pages_cut(s.free, s.cache, i32(0, 16))
    assert int(s.free[0]) == 2   # the one that was free and the sequence's one page, not the six that it never had
    granted, slots = i32(-9, -9), torch.empty(2, 60, dtype=torch.int64, device="cuda")
    pages_take(s.free, s.cache, i32(0, 48), granted, slots=slots)
    assert granted.tolist() == [0, 0]
    pages_take(s.free, s.cache, i32(0, 32), granted, slots=slots)
    assert granted.tolist() == [0, 32] and int(slots[1, :32].min()) >= 0


def test_a_stack_of_other_pages_of_the_pool():
    """Page numbers may lie beyond the stack's room: they are pages as long as the pool has them."""
    from amdgpu_rustdsl_b200 import pages_cut, pages_take
    s = P.State([0, 0], 16, 4, 20)
    free = torch.tensor([3, 0, 0, 0, 19, 17, 18], dtype=torch.int32, device="cuda")
    before, granted = free.clone(), torch.zeros(2, dtype=torch.int32, device="cuda")
    pages_take(free, s.cache, torch.tensor([20, 5], dtype=torch.int32, device="cuda"), granted)
    assert granted.tolist() == [20, 5] and s.cache.table.tolist() == [[18, 17, -1, -1], [19, -1, -1, -1]]
    pages_cut(free, s.cache, torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert torch.equal(free, before)
