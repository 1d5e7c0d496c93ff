"""Python entry of the operators around a key/value cache held in 4 bits (head dim 128): append, read back, attention, eviction.

The cache is the caller's memory: a pool of pages (``kv4_pool``), a page table and lengths, held together by a ``Kv4Cache``. Per layer and step a server
raises the lengths, appends the new tokens and attends:

    cache = Kv4Cache(kv4_pool(pages, kv_heads, device=dev), table, lengths)   # once per layer
    lengths += new_tokens
    kv4_append(cache, k, v)
    fmha_fwd_kv4(q, cache, out, weights=w, weights_in=w)                      # w: what eviction goes by, None where nobody asks
    kv4_evict(cache, w, smaller, keep=1024, recent=128)                       # when the pages run out

PyTorch owns memory and streams only; every call goes to the sm_100a kernels behind the C ABI of ``include/fmha_kv4_abi.h``. Calls run on torch's current stream of
the cache's device (or ``stream``, a raw handle) and do not wait for it. Scratch memory is kept per stream; several threads may make calls on one. In a graph that ``torch.cuda.graph`` captures
it is the graph's own. Wrong arguments raise ``ValueError``.
"""
from __future__ import annotations

import ctypes as C
import math
import threading

from . import _abi
from .ops import _raw_stream, _ws, _ws_lock

D = 128
TOKEN_BYTES = 136   # a token's K and V of one KV head: 2 x (64 code bytes + 4 scale bytes)
PAGE_SIZES = (16, 32, 64, 128)


def kv4_pool(pages, kv_heads, page=64, device="cuda"):
    """An empty pool for ``pages`` pages of ``page`` tokens: uint8 [pages, kv_heads, 136 * page]."""
    import torch
    if page not in PAGE_SIZES:
        raise ValueError(f"kv4_pool: pages hold 16, 32, 64 or 128 tokens, not {page}")
    return torch.zeros((pages, kv_heads, TOKEN_BYTES * page), dtype=torch.uint8, device=device)


class PagedCache:
    """Views of the caller's pool, table and lengths as the C struct: what the caches of 4 and of 8 bits have in common."""
    __slots__ = ("pool", "table", "lengths", "page", "B", "HK", "capacity", "device", "c")
    TOKEN_BYTES = 0   # of a token and KV head

    def __init__(self, pool, table, lengths):
        import torch
        who, token = type(self).__name__, self.TOKEN_BYTES
        if pool.dtype != torch.uint8 or pool.dim() != 3 or pool.shape[2] % token or pool.shape[2] // token not in PAGE_SIZES:
            raise ValueError(f"{who}: pool must be uint8 [pages, KV heads, {token} * page] with pages of 16, 32, 64 or 128 tokens")
        if table.dtype != torch.int32 or table.dim() != 2 or lengths.dtype != torch.int32 or tuple(lengths.shape) != (table.shape[0],):
            raise ValueError(f"{who}: table must be int32 [B, width] and lengths int32 [B]")
        for name, t in (("pool", pool), ("table", table), ("lengths", lengths)):
            if not t.is_cuda or t.device != pool.device or not t.is_contiguous() or t.numel() == 0:
                raise ValueError(f"{who}: {name} must be a contiguous CUDA tensor on the pool's device with something in it")
        if pool.data_ptr() % 16:
            raise ValueError(f"{who}: pool must start on a 16-byte boundary")
        self.pool, self.table, self.lengths, self.device = pool, table, lengths, pool.device
        self.page, self.HK, self.B = pool.shape[2] // token, pool.shape[1], table.shape[0]
        self.capacity = table.shape[1] * self.page   # tokens that a sequence has room for
        self.c = _abi.Kv4CacheArgs(pool.data_ptr(), table.data_ptr(), lengths.data_ptr(), pool.shape[0], self.B, self.HK, self.page, table.shape[1])


class Kv4Cache(PagedCache):
    """A paged cache of MXFP4 keys and values: views of the caller's tensors, nothing of its own.

    pool     uint8 [pages, HK, 136 * page], page 16, 32, 64 or 128 (``kv4_pool``)
    table    int32 [B, width]: pages of a sequence's tokens in order; entries behind its length are never looked at
    lengths  int32 [B]: tokens of each sequence, new ones included, read by the kernels when they run

    The tensors may be written between calls (on the stream of the calls), not replaced.
    """
    __slots__ = ()
    TOKEN_BYTES = TOKEN_BYTES


def _rows(who, name, x, cache, S=None, heads=None):
    """bf16 [B, S, heads, 128] with a dense last dimension as the C struct."""
    import torch
    shape = x.shape
    b, s, h, d = shape if len(shape) == 4 else (0, 0, 0, 0)
    if x.dtype != torch.bfloat16 or b != cache.B or d != D or (S is not None and s != S) or (heads is not None and h != heads):
        raise ValueError(f"{who}: {name} must be bf16 [{cache.B}, {'S' if S is None else S}, {'H' if heads is None else heads}, 128], not {x.dtype} {tuple(shape)}")
    sb, ss, sh, sd = x.stride()
    ptr = x.data_ptr()
    if x.device != cache.device or sd != 1 or (sb | ss | sh) & 7 or ptr & 15:
        raise ValueError(f"{who}: {name} must be on the cache's device, its last dimension dense, its start and its strides multiples of 16 bytes")
    if s > 0x7FFFFFFF:   # (a stride of 0 makes as many rows as you like; the library counts them in 32 bits)
        raise ValueError(f"{who}: {name} has {s} rows, more than 2^31")
    return _abi.Kv4Rows(ptr, sb, ss, sh)


def _i32(who, name, x, cache, shape):
    import torch
    if x is None:
        return None
    if x.dtype != torch.int32 or x.shape != shape or x.device != cache.device or not x.is_contiguous():
        raise ValueError(f"{who}: {name} must be a contiguous int32 tensor of shape {shape} on the cache's device")
    return x.data_ptr()


def _f32(who, name, x, cache, at_least):
    """f32 [B, HK, width >= at_least]"""
    import torch
    if x.dtype != torch.float32 or x.dim() != 3 or x.shape[0] != cache.B or x.shape[1] != cache.HK or x.shape[2] < at_least or x.device != cache.device or not x.is_contiguous():
        raise ValueError(f"{who}: {name} must be a contiguous f32 tensor [{cache.B}, {cache.HK}, {at_least} or more] on the cache's device")
    return x.data_ptr()


class _Errors(threading.local):
    """A thread's buffer for the library's messages."""

    def __init__(self):
        self.text = C.create_string_buffer(256)


_errors = _Errors()


def _check(who, rc):
    if rc > 0:
        raise ValueError(f"{who}: {_errors.text.value.decode()}")
    if rc < 0:
        raise RuntimeError(f"{who} failed with code {rc}: {_errors.text.value.decode()}")


def _call(torch, cache, stream, fn, *args):
    """fn(*args, stream, err, cap) with the cache's device current."""
    if torch.cuda.current_device() == (cache.device.index or 0):
        return fn(*args, stream, _errors.text, 256)
    with torch.cuda.device(cache.device):
        return fn(*args, stream, _errors.text, 256)


def _is_kv4(who, cache, name="cache"):
    if not isinstance(cache, Kv4Cache):   # (the 8-bit cache has the same fields, and other contents)
        raise ValueError(f"{who}: {name} must be a Kv4Cache, not {type(cache).__name__}")


def kv4_append(cache, k, v, *, counts=None, stream=None):
    """Rounds the newest tokens' keys and values into the cache: k, v bf16 [B, S, HK, 128] (slices of a wider projection are fine).

    Row i of sequence b becomes token ``lengths[b] - n + i``, with n = S, or ``counts[b]`` (int32 [B]) of the S rows where the sequences have different numbers of
    new tokens, and never more than the length. The lengths are the caller's to raise, before this call. Per 32 elements one E8M0 scale,
    floor(log2 of the largest) - 2, elements e2m1 rounded to nearest, ties to even, saturating at 6 times the scale; a block with Inf or NaN reads as NaN."""
    import torch
    _is_kv4("kv4_append", cache)
    lib = _abi.load()
    rk = _rows("kv4_append", "k", k, cache, heads=cache.HK)
    rv = _rows("kv4_append", "v", v, cache, k.shape[1], cache.HK)
    n = _i32("kv4_append", "counts", counts, cache, (cache.B,))
    raw = stream if stream is not None else _raw_stream(torch, cache.device)
    rc = _call(torch, cache, raw, lib.fmha_kv4_append, cache.c, rk, rv, k.shape[1], n)
    if rc:
        _check("kv4_append", rc)


def kv4_read(cache, k, v, *, last=False, counts=None, stream=None):
    """The values that the cache holds, exact in bf16, into k, v [B, S, HK, 128]: tokens 0 .. S - 1, or with ``last`` the newest ones, row for row as
    ``kv4_append`` took them (``counts`` as there). Rows that stand for no token become zeros."""
    import torch
    _is_kv4("kv4_read", cache)
    lib = _abi.load()
    rk = _rows("kv4_read", "k", k, cache, heads=cache.HK)
    rv = _rows("kv4_read", "v", v, cache, k.shape[1], cache.HK)
    n = _i32("kv4_read", "counts", counts, cache, (cache.B,))
    raw = stream if stream is not None else _raw_stream(torch, cache.device)
    rc = _call(torch, cache, raw, lib.fmha_kv4_read, cache.c, rk, rv, k.shape[1], 1 if last else 0, n)
    if rc:
        _check("kv4_read", rc)


def fmha_fwd_kv4(q, cache, out, *, causal=True, counts=None, scale=None, lse=None, weights=None, weights_in=None, stream=None):
    """Attention over the cache: ``out = softmax(scale q k^T) v``, q bf16 [B, S, H, 128] (strided), out bf16 [B, S, H, 128] (packed), H = 1 to 16 times the KV heads.

    out         shares no memory with q; or it is q, packed, without ``weights`` or with at most 8 rows (S times H / HK) of a KV head
    causal      the rows are the sequences' newest tokens (``counts`` as in ``kv4_append``): row i of n sees the tokens up to ``lengths[b] - n + i``. Without it every row
                sees all tokens. Rows beyond n, and rows that see nothing, are zeros.
    scale       1 / sqrt(128) where not given
    lse         f32 [B, H, S]: natural log-sum-exps, -inf for rows that see nothing
    weights     f32 [B, HK, capacity or more]: for each token t below the length, the softmax weight that it received from the rows and the query heads of its KV head,
                plus ``weights_in`` there (the same shape; the same tensor, or one that shares no memory with it) where given; with ``causal`` the n newest tokens start from nothing. Nothing is
                written behind the length. The sums are the same bits every time.
    """
    import torch
    _is_kv4("fmha_fwd_kv4", cache)
    lib = _abi.load()
    a = _abi.Kv4AttendArgs()
    a.q = _rows("fmha_fwd_kv4", "q", q, cache)
    _, S, H, _ = q.shape
    if out.dtype != torch.bfloat16 or out.shape != q.shape or not out.is_contiguous() or out.device != cache.device:
        raise ValueError(f"fmha_fwd_kv4: out must be a contiguous bf16 tensor of q's shape {tuple(q.shape)} on the cache's device")
    a.out, a.S, a.H, a.causal = out.data_ptr(), S, H, 1 if causal else 0
    a.scale = 1.0 / math.sqrt(D) if scale is None else scale
    a.counts = _i32("fmha_fwd_kv4", "counts", counts, cache, (cache.B,))
    if lse is not None:
        if lse.dtype != torch.float32 or tuple(lse.shape) != (cache.B, H, S) or not lse.is_contiguous() or lse.device != cache.device:
            raise ValueError(f"fmha_fwd_kv4: lse must be a contiguous f32 tensor of shape {(cache.B, H, S)} on the cache's device")
        a.lse = lse.data_ptr()
    if weights is not None:
        a.weights, a.weights_width = _f32("fmha_fwd_kv4", "weights", weights, cache, cache.capacity), weights.shape[2]
        if weights_in is not None:
            if weights_in.shape != weights.shape:
                raise ValueError("fmha_fwd_kv4: weights_in must have the shape of weights")
            a.weights_in = _f32("fmha_fwd_kv4", "weights_in", weights_in, cache, cache.capacity)
    elif weights_in is not None:
        raise ValueError("fmha_fwd_kv4: weights_in without weights")
    raw = stream if stream is not None else _raw_stream(torch, cache.device)
    nbytes = lib.fmha_kv4_attend_workspace(cache.c, a)
    with _ws_lock(cache.device, raw):
        ws = _ws("kv4", nbytes, cache.device, raw)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        rc = _call(torch, cache, raw, lib.fmha_kv4_attend, cache.c, a)
    if rc:
        _check("fmha_fwd_kv4", rc)


def kv4_evict(cache, weights, into, *, keep, recent=0, first=0, kept=None, weights_out=None, stream=None):
    """Cuts every sequence to ``keep`` tokens per KV head and packs them, in order, into ``into``, a ``Kv4Cache`` whose pages are not read by ``cache`` (the pool may be
    the same); its lengths become min(length, keep).

    The first ``first`` and the last ``recent`` tokens stay, and of the others those with the greatest ``weights`` (f32 [B, HK, capacity or more], as ``fmha_fwd_kv4``
    accumulates them); among equals the earlier ones, and NaN counts as more than any number. Different heads keep different tokens.
    kept         int32 [B, HK, keep]: the positions that stayed, ascending, -1 behind them
    weights_out  f32 [B, HK, keep or more]: their weights, for the next eviction; nothing is written behind the new length. Another tensor than ``weights``, whose
                 memory it must not share.
    """
    import torch
    _is_kv4("kv4_evict", cache)
    _is_kv4("kv4_evict", into, "into")
    lib = _abi.load()
    a = _abi.Kv4EvictArgs()
    if into.device != cache.device:
        raise ValueError("kv4_evict: into must be on the cache's device")
    a.weights, a.weights_width = _f32("kv4_evict", "weights", weights, cache, cache.capacity), weights.shape[2]
    if not 1 <= keep <= into.capacity or recent < 0 or first < 0 or first + recent > keep:   # (here, in numbers of any size: the struct's have 32 bits)
        raise ValueError(f"kv4_evict: keep must be 1 to the {into.capacity} tokens that into has room for, recent and first not negative and no more than keep together")
    a.keep, a.recent, a.first = keep, recent, first
    raw = stream if stream is not None else _raw_stream(torch, cache.device)
    a.kept = _i32("kv4_evict", "kept", kept, cache, (cache.B, cache.HK, keep))
    if weights_out is not None:
        a.weights_out, a.weights_out_width = _f32("kv4_evict", "weights_out", weights_out, cache, keep), weights_out.shape[2]
    if kept is not None:
        rc = _call(torch, cache, raw, lib.fmha_kv4_evict, cache.c, into.c, a)
    else:
        with _ws_lock(cache.device, raw):
            scratch = _ws("kv4_kept", 4 * cache.B * cache.HK * keep, cache.device, raw)
            a.kept = scratch.data_ptr()
            rc = _call(torch, cache, raw, lib.fmha_kv4_evict, cache.c, into.c, a)
    if rc:
        _check("kv4_evict", rc)
