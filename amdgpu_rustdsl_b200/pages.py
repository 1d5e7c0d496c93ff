"""Python entry of the bookkeeping of a paged cache's pages on the device: which pages the new tokens of a step go to, how long the sequences are then, where each token stands.

    free = pages_stack(pages, device=dev)                                                # int32 [4 + pages]: all pages are free
    pages_take(free, cache, counts, granted, positions=positions, slots=slots)           # a step's new tokens: table, lengths, positions
    pages_cut(free, cache, keep)                                                         # tokens that go: drafts that were not accepted, sequences that are over

``cache`` is a ``Kv4Cache`` or ``Kv8Cache``, of which only table, lengths and page size are looked at: layers that share a table need one call. Nothing is read back: a server can go on
enqueueing, and look at ``granted`` when it likes. The calls go to the sm_100a kernels behind the C ABI of ``include/fmha_pages_abi.h``, run on torch's current stream of the cache's
device (or ``stream``, a raw handle) and do not wait for it. Wrong arguments raise ``ValueError``.
"""
from __future__ import annotations

from . import _abi
from .kv4 import PagedCache, _call, _check, _i32
from .ops import _raw_stream


def pages_stack(pages, device="cuda"):
    """A stack of ``pages`` free pages, 0 on top: int32 [4 + pages], the first word how many are free."""
    import torch
    if not 1 <= pages <= 0x7FFFFFF0:
        raise ValueError(f"pages_stack: 1 to 2^31 - 16 pages, not {pages}")
    return torch.cat([torch.tensor([pages, 0, 0, 0], dtype=torch.int32), torch.arange(pages - 1, -1, -1, dtype=torch.int32)]).to(device)


def _pages(who, free, cache):
    import torch
    if not isinstance(cache, PagedCache):
        raise ValueError(f"{who}: cache must be a Kv4Cache or a Kv8Cache, not {type(cache).__name__}")
    if free.dtype != torch.int32 or free.dim() != 1 or free.shape[0] < 5 or not free.is_contiguous() or free.device != cache.device:
        raise ValueError(f"{who}: free must be a contiguous int32 tensor [4 + pages] on the cache's device")
    return _abi.PagesArgs(free.data_ptr(), cache.c.table, cache.c.lengths, free.shape[0] - 4, cache.B, cache.page, cache.table.shape[1])


def pages_take(free, cache, counts, granted, *, positions=None, slots=None, starts=None, stream=None):
    """Makes room for ``counts[b]`` (int32 [B]) new tokens of each sequence: pages go from the stack to the table, in the order of the sequences, and the lengths grow.

    A sequence is granted all of its tokens or none: none where its row of the table has no room for them, or where it needs pages and those needed by it and the sequences
    in front of it are more than are free.

    granted    int32 [B]: counts[b] or 0; what ``kv8_append`` and the attention take as ``counts``
    positions  int32 or int64 [B, S]: of row i < granted[b] the token it becomes, the length before plus i; -1 in other rows. (``counts`` may go beyond S, the rows do not: tokens without a row are
               whoever writes them's to look after)
    slots      int64 [B, S]: page number times tokens of a page, plus the place within it, of that token; -1 in other rows
    starts     int32 [B + 1]: the sums of granted in front of each sequence, and of all; for stacks of less than 2^31 tokens
    """
    import torch
    lib = _abi.load()
    p = _pages("pages_take", free, cache)
    if counts is None or granted is None:
        raise ValueError("pages_take: counts and granted must be given")
    n, g = _i32("pages_take", "counts", counts, cache, (cache.B,)), _i32("pages_take", "granted", granted, cache, (cache.B,))
    S = 0
    for name, x, kinds in (("positions", positions, (torch.int32, torch.int64)), ("slots", slots, (torch.int64,))):
        if x is None:
            continue
        if x.dtype not in kinds or x.dim() != 2 or x.shape[0] != cache.B or (S and x.shape[1] != S) or x.device != cache.device or not x.is_contiguous():
            raise ValueError(f"pages_take: {name} must be a contiguous {" or ".join(map(str, kinds))} tensor [{cache.B}, S] on the cache's device, positions and slots with the same S")
        S = x.shape[1]
    if S > 0x7FFFFFFF:
        raise ValueError(f"pages_take: {S} rows, more than 2^31")
    if positions is not None and slots is not None and positions.shape != slots.shape:
        raise ValueError("pages_take: positions and slots must have the same S")
    s = _i32("pages_take", "starts", starts, cache, (cache.B + 1,))
    raw = stream if stream is not None else _raw_stream(torch, cache.device)
    rc = _call(torch, cache, raw, lib.fmha_pages_take, p, n, g, None if positions is None else positions.data_ptr(), positions is not None and positions.dtype == torch.int64, None if slots is None else slots.data_ptr(), s, S)
    if rc:
        _check("pages_take", rc)


def pages_cut(free, cache, keep, *, stream=None):
    """Cuts every sequence to ``keep[b]`` (int32 [B]) tokens, if it has more; its pages without tokens go back to the stack, and their entries in the table become -1.

    A cut to the lengths before a ``pages_take`` leaves stack, table and lengths as they were before it. ``keep`` of 0 ends a sequence."""
    import torch
    lib = _abi.load()
    p = _pages("pages_cut", free, cache)
    if keep is None:
        raise ValueError("pages_cut: keep must be given")
    k = _i32("pages_cut", "keep", keep, cache, (cache.B,))
    raw = stream if stream is not None else _raw_stream(torch, cache.device)
    rc = _call(torch, cache, raw, lib.fmha_pages_cut, p, k)
    if rc:
        _check("pages_cut", rc)
