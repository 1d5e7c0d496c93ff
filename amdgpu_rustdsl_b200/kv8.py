"""Python entry of the operators around a key/value cache held in 8 bits (head dim 128): append, read back, attention.

Beside the 4-bit cache of ``kv4``, and used like it, for models that 4 bits are too few for: e4m3 elements with one power of two for 16 tokens of a head, 257 bytes per
token and KV head in place of 512.

    cache = Kv8Cache(kv8_pool(pages, kv_heads, device=dev), table, lengths)   # once per layer
    pages_take(free, cache, counts, granted, positions=positions)              # once per step: pages, lengths, positions
    rope_rotate(rope, q, positions, y=k)                                       # per layer
    kv8_append(cache, k, v, counts=granted)
    fmha_fwd_kv8(q, cache, out, counts=granted)

PyTorch owns memory and streams only; every call goes to the sm_100a kernels behind the C ABI of ``include/fmha_kv8_abi.h``. Calls run on torch's current stream of
the cache's device (or ``stream``, a raw handle) and do not wait for it. Scratch memory is kept per stream; several threads may make calls on one. In a graph that
``torch.cuda.graph`` captures it is the graph's own. Wrong arguments raise ``ValueError``.
"""
from __future__ import annotations

import math

from . import _abi
from .kv4 import D, PAGE_SIZES, PagedCache, _call, _check, _i32, _rows
from .ops import _raw_stream, _ws, _ws_lock

TOKEN_BYTES = 257   # a token's K and V of one KV head: 2 x 128 codes, and its part of the 16 bytes that a block of 16 tokens has for scales and masks


def kv8_pool(pages, kv_heads, page=64, device="cuda"):
    """A pool for ``pages`` pages of ``page`` tokens: uint8 [pages, kv_heads, 257 * page]."""
    import torch
    if page not in PAGE_SIZES:
        raise ValueError(f"kv8_pool: pages hold 16, 32, 64 or 128 tokens, not {page}")
    return torch.zeros((pages, kv_heads, TOKEN_BYTES * page), dtype=torch.uint8, device=device)


class Kv8Cache(PagedCache):
    """A paged cache of e4m3 keys and values with a scale per 16 tokens and head: views of the caller's tensors, nothing of its own.

    pool     uint8 [pages, HK, 257 * page], page 16, 32, 64 or 128 (``kv8_pool``)
    table    int32 [B, width]: pages of a sequence's tokens in order; entries behind its length are never looked at
    lengths  int32 [B]: tokens of each sequence, new ones included, read by the kernels when they run

    The tensors may be written between calls (on the stream of the calls), not replaced.
    """
    __slots__ = ()
    TOKEN_BYTES = TOKEN_BYTES


def _is_kv8(who, cache):
    if not isinstance(cache, Kv8Cache):
        raise ValueError(f"{who}: cache must be a Kv8Cache, not {type(cache).__name__}")


def kv8_append(cache, k, v, *, counts=None, stream=None):
    """Rounds the newest tokens' keys and values into the cache: k, v bf16 [B, S, HK, 128] (slices of a wider projection are fine).

    Row i of sequence b becomes token ``lengths[b] - n + i``, with n = S, or ``counts[b]`` (int32 [B]) of the S rows where the sequences have different numbers of
    new tokens, and never more than the length. The lengths are the caller's to raise, before this call (``pages_take`` does). Per 16 tokens and head one scale for K
    and one for V, the smallest power of two that leaves no element above 448 of it; elements e4m3, rounded to nearest, ties to even. A block that has tokens already keeps
    its scale, or its tokens' codes move to a larger one, which costs bits only below 2^-6 of that. (Sequences may share pages that are full, as long as nobody takes those back:
    ``pages_cut`` does not count their users. A page that one of them still fills is its own.)
    A token with Inf or NaN in its K (V) reads as NaN there throughout."""
    import torch
    _is_kv8("kv8_append", cache)
    lib = _abi.load()
    rk = _rows("kv8_append", "k", k, cache, heads=cache.HK)
    rv = _rows("kv8_append", "v", v, cache, k.shape[1], cache.HK)
    n = _i32("kv8_append", "counts", counts, cache, (cache.B,))
    raw = stream if stream is not None else _raw_stream(torch, cache.device)
    rc = _call(torch, cache, raw, lib.fmha_kv8_append, cache.c, rk, rv, k.shape[1], n)
    if rc:
        _check("kv8_append", rc)


def kv8_read(cache, k, v, *, last=False, counts=None, stream=None):
    """The values that the cache holds, exact in bf16, into k, v [B, S, HK, 128]: tokens 0 .. S - 1, or with ``last`` the newest ones, row for row as
    ``kv8_append`` took them (``counts`` as there). Rows that stand for no token become zeros."""
    import torch
    _is_kv8("kv8_read", cache)
    lib = _abi.load()
    rk = _rows("kv8_read", "k", k, cache, heads=cache.HK)
    rv = _rows("kv8_read", "v", v, cache, k.shape[1], cache.HK)
    n = _i32("kv8_read", "counts", counts, cache, (cache.B,))
    raw = stream if stream is not None else _raw_stream(torch, cache.device)
    rc = _call(torch, cache, raw, lib.fmha_kv8_read, cache.c, rk, rv, k.shape[1], 1 if last else 0, n)
    if rc:
        _check("kv8_read", rc)


def fmha_fwd_kv8(q, cache, out, *, causal=True, counts=None, scale=None, lse=None, stream=None):
    """Attention over the cache: ``out = softmax(scale q k^T) v``, q bf16 [B, S, H, 128] (strided), out bf16 [B, S, H, 128] (packed), H = 1 to 16 times the KV heads.

    out         shares no memory with q; or it is q, packed
    causal      the rows are the sequences' newest tokens (``counts`` as in ``kv8_append``): row i of n sees the tokens up to ``lengths[b] - n + i``. Without it every row
                sees all tokens. Rows beyond n, and rows that see nothing, are zeros.
    scale       1 / sqrt(128) where not given
    lse         f32 [B, H, S]: natural log-sum-exps, -inf for rows that see nothing
    """
    import torch
    _is_kv8("fmha_fwd_kv8", cache)
    lib = _abi.load()
    a = _abi.Kv8AttendArgs()
    a.q = _rows("fmha_fwd_kv8", "q", q, cache)
    _, S, H, _ = q.shape
    if out.dtype != torch.bfloat16 or out.shape != q.shape or not out.is_contiguous() or out.device != cache.device:
        raise ValueError(f"fmha_fwd_kv8: out must be a contiguous bf16 tensor of q's shape {tuple(q.shape)} on the cache's device")
    a.out, a.S, a.H, a.causal = out.data_ptr(), S, H, 1 if causal else 0
    a.scale = 1.0 / math.sqrt(D) if scale is None else scale
    a.counts = _i32("fmha_fwd_kv8", "counts", counts, cache, (cache.B,))
    if lse is not None:
        if lse.dtype != torch.float32 or tuple(lse.shape) != (cache.B, H, S) or not lse.is_contiguous() or lse.device != cache.device:
            raise ValueError(f"fmha_fwd_kv8: lse must be a contiguous f32 tensor of shape {(cache.B, H, S)} on the cache's device")
        a.lse = lse.data_ptr()
    raw = stream if stream is not None else _raw_stream(torch, cache.device)
    nbytes = lib.fmha_kv8_attend_workspace(cache.c, a)
    with _ws_lock(cache.device, raw):
        ws = _ws("kv8", nbytes, cache.device, raw)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        rc = _call(torch, cache, raw, lib.fmha_kv8_attend, cache.c, a)
    if rc:
        _check("fmha_fwd_kv8", rc)
