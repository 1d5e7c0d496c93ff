"""Python entry of the bookkeeping of a paged cache's pages on the device: which pages the new tokens of a step go to, how long the sequences are then, where each token stands.

    free = pages_stack(pages, device=dev)                                                # int32 [4 + pages]: all pages are free
    pages_take(free, cache, counts, granted, positions=positions, slots=slots)           # a step's new tokens: table, lengths, positions
    pages_cut(free, cache, keep)                                                         # tokens that go: drafts that were not accepted, sequences that are over

``cache`` is a ``Kv4Cache`` or ``Kv8Cache``, of which only table, lengths and page size are looked at: layers that share a table need one call. Nothing is read back: a server can go on
enqueueing, and look at ``granted`` when it likes. The calls go to the sm_100a kernels behind the C ABI of ``include/fmha_pages_abi.h``, run on torch's current stream of the cache's
device (or ``stream``, a raw handle) and do not wait for it. Wrong arguments raise ``ValueError``.
"""
from __future__ import annotations

import ctypes as C
import struct

from . import _abi
from .kv4 import PagedCache, _call, _check, _i32
from .ops import _raw_stream


_ARGS = struct.Struct("@3Q5I4x").pack   # fmha_pages, as bytes: half the time that a ctypes structure takes
assert struct.calcsize("@3Q5I4x") == C.sizeof(_abi.PagesArgs)
_entries = {}


def _entry(name, *kinds):
    """The C entry with its first argument as bytes."""
    entry = _abi.load()[name]
    entry.restype, entry.argtypes = C.c_int, [C.c_char_p, *kinds, C.c_void_p, C.c_char_p, C.c_size_t]
    _entries[name] = entry
    return entry


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
    shape = free.shape
    if free.dtype != torch.int32 or len(shape) != 1 or shape[0] < 5 or not free.is_contiguous() or free.device != cache.device:
        raise ValueError(f"{who}: free must be a contiguous int32 tensor [4 + pages] on the cache's device")
    pages = shape[0] - 4
    if pages > 0x7FFFFFFF:   # (here, in numbers of any size)
        raise ValueError(f"{who}: a stack of {pages} pages, more than 2^31")
    c = cache.c
    return _ARGS(free.data_ptr(), c.table, c.lengths, pages, c.B, c.page, c.table_width, c.pages)


def _map(name, x, kind, cache):
    """S of a map's [B, S]."""
    shape = x.shape
    if not kind or len(shape) != 2 or shape[0] != cache.B or x.device != cache.device or not x.is_contiguous():
        raise ValueError(f"pages_take: {name} must be a contiguous {'torch.int32 or torch.int64' if name == 'positions' else 'torch.int64'} tensor [{cache.B}, S] on the cache's device")
    return shape[1]


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
    p = _pages("pages_take", free, cache)
    if counts is None or granted is None:
        raise ValueError("pages_take: counts and granted must be given")
    n, g = _i32("pages_take", "counts", counts, cache, (cache.B,)), _i32("pages_take", "granted", granted, cache, (cache.B,))
    S, wide, at_positions, at_slots = 0, False, None, None
    if positions is not None:
        wide = positions.dtype == torch.int64
        S, at_positions = _map("positions", positions, wide or positions.dtype == torch.int32, cache), positions.data_ptr()
    if slots is not None:
        rows, at_slots = _map("slots", slots, slots.dtype == torch.int64, cache), slots.data_ptr()
        if positions is not None and rows != S:
            raise ValueError("pages_take: positions and slots must have the same S")
        S = rows
    if S > 0x7FFFFFFF:
        raise ValueError(f"pages_take: {S} rows, more than 2^31")
    s = _i32("pages_take", "starts", starts, cache, (cache.B + 1,))
    raw = stream if stream is not None else _raw_stream(torch, cache.device)
    take = _entries.get("fmha_pages_take") or _entry("fmha_pages_take", C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_uint32)
    rc = _call(torch, cache, raw, take, p, n, g, at_positions, wide, at_slots, s, S)
    if rc:
        _check("pages_take", rc)


def pages_cut(free, cache, keep, *, stream=None):
    """Cuts every sequence to ``keep[b]`` (int32 [B]) tokens, if it has more; its pages without tokens go back to the stack, and their entries in the table become -1. (Entries that
    name no page of the pool give none back.)

    A cut to the lengths before a ``pages_take`` leaves stack, table and lengths as they were before it. ``keep`` of 0 ends a sequence.

    Nobody counts a page's users: every page behind ``keep`` is handed out again. Pages that other sequences hold too (a prefix in common) have to lie in front of ``keep``: such a sequence ends with
    ``keep`` at the prefix's end, and the prefix's pages are the caller's to give back when nobody holds them any more."""
    import torch
    p = _pages("pages_cut", free, cache)
    if keep is None:
        raise ValueError("pages_cut: keep must be given")
    k = _i32("pages_cut", "keep", keep, cache, (cache.B,))
    raw = stream if stream is not None else _raw_stream(torch, cache.device)
    rc = _call(torch, cache, raw, _entries.get("fmha_pages_cut") or _entry("fmha_pages_cut", C.c_void_p), p, k)
    if rc:
        _check("pages_cut", rc)
