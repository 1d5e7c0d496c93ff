"""The bookkeeping of pages without a GPU: wrong arguments are refused with a message before anything is launched or read."""
import ctypes as C

import pytest
import torch

FAKE = 1 << 20   # an aligned address that nothing follows: every call here is refused


def _pages(abi, **change):
    p = abi.PagesArgs(free=FAKE, table=2 * FAKE, lengths=3 * FAKE, pages=100, B=4, page=16, table_width=8)
    for k, v in change.items():
        setattr(p, k, v)
    return p


def _take(abi, p, counts=4 * FAKE, granted=5 * FAKE, positions=6 * FAKE, slots=7 * FAKE, starts=8 * FAKE, S=3, wide=0):
    err = C.create_string_buffer(256)
    return abi.load().fmha_pages_take(p, counts, granted, positions, wide, slots, starts, S, None, err, 256), err.value.decode()


def _cut(abi, p, keep=4 * FAKE):
    err = C.create_string_buffer(256)
    return abi.load().fmha_pages_cut(p, keep, None, err, 256), err.value.decode()


@pytest.mark.parametrize("change,message", [({"free": None}, "must be given"), ({"table": None}, "must be given"), ({"lengths": None}, "must be given"), ({"page": 48}, "16, 32, 64 or 128"), ({"B": 0}, "no sequences"),
                                            ({"pages": 0}, "no sequences"), ({"table_width": 0}, "no sequences"), ({"pages": 0x7FFFFFFF}, "2^31"), ({"table_width": 1 << 28}, "2^31"), ({"B": (1 << 30) + 1}, "2^30"),
                                            ({"lengths": 2 * FAKE + 4}, "share memory"), ({"table": FAKE + 8}, "share memory")])
def test_bad_pages_are_refused(abi, change, message):
    for call in (_take, _cut):
        rc, err = call(abi, _pages(abi, **change))
        assert rc == 6 and message in err


@pytest.mark.parametrize("change,message", [({"counts": None}, "must be given"), ({"granted": None}, "must be given"), ({"granted": 4 * FAKE}, "granted must not share"), ({"positions": 5 * FAKE + 8}, "granted must not share"),
                                            ({"slots": 6 * FAKE + 40}, "positions must not share"), ({"starts": 7 * FAKE + 90}, "slots must not share"), ({"starts": 4 * FAKE + 8}, "counts"),
                                            ({"positions": FAKE + 400}, "the stack"), ({"slots": 2 * FAKE + 100}, "the table"), ({"starts": 3 * FAKE + 12}, "the lengths"), ({"S": 1 << 29}, "2^30"), ({"slots": 6 * FAKE + 48, "wide": 1}, "positions must not share")])
def test_bad_takes_are_refused(abi, change, message):
    rc, err = _take(abi, _pages(abi), **change)
    assert rc == 6 and message in err, err


def test_bad_cuts_are_refused(abi):
    for keep, message in ((None, "must be given"), (3 * FAKE, "lengths must not share memory with keep"), (FAKE + 100, "stack"), (2 * FAKE, "table")):
        rc, err = _cut(abi, _pages(abi), keep)
        assert rc == 6 and message in err, err


def test_a_stack_of_all_pages():
    from amdgpu_rustdsl_b200 import pages_stack
    assert pages_stack(3, device="cpu").tolist() == [3, 0, 0, 0, 2, 1, 0]
    with pytest.raises(ValueError, match="pages_stack"):
        pages_stack(0, device="cpu")


def test_only_caches_have_pages():
    from amdgpu_rustdsl_b200 import pages_cut, pages_stack, pages_take
    one = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: pages_take(pages_stack(3, device="cpu"), one, one, one), lambda: pages_cut(pages_stack(3, device="cpu"), None, one)):
        with pytest.raises(ValueError, match="Kv4Cache or a Kv8Cache"):
            call()


def test_starts_that_do_not_fit_are_refused(abi):
    """Sums of granted tokens are 32 bits: a stack of 2^27 pages of 16 tokens is too many for them (and is taken without starts: the refusal is the next one)."""
    rc, err = _take(abi, _pages(abi, pages=1 << 27, free=1 << 40), starts=8 * FAKE)
    assert rc == 6 and "starts" in err
    rc, err = _take(abi, _pages(abi, pages=1 << 27, free=1 << 40), starts=None, S=1 << 29)
    assert rc == 6 and "2^30 rows" in err
