"""Generation with a 4-bit cache of bounded size: prompts go in, tokens come out, and whenever the room runs out every head drops what it looked at least.

    python -m amdgpu_rustdsl_b200.kv4_example [--sequences 16 --heads 32 --kv-heads 8 --prompt 2048 --steps 3000 --room 4096 --keep 2048]

runs one attention layer on random projections (there is no model here) and prints what a step of each kind takes.
"""
from __future__ import annotations

import argparse

from .kv4 import Kv4Cache, fmha_fwd_kv4, kv4_append, kv4_evict, kv4_pool


class BoundedCache:
    """A layer's cache of ``room`` tokens per sequence that is cut to ``keep`` when it is full: two sets of pages of one pool, one of which an eviction fills from the other.

    step(q, k, v, out, counts) takes the new tokens' projections (bf16 [B, S, heads, 128], rotated already: tokens keep the positions they were given when others
    before them go) and leaves their attention in ``out``. ``first`` and ``recent`` tokens always stay."""

    def __init__(self, sequences, kv_heads, room, keep, recent=64, first=4, page=64, device="cuda"):
        import torch
        width = -(-room // page)
        if not first + recent <= keep < width * page:
            raise ValueError("BoundedCache: keep must be less than the room and not less than first and recent together")
        pool = kv4_pool(2 * sequences * width, kv_heads, page, device)
        tables = torch.arange(2 * sequences * width, dtype=torch.int32, device=device).view(2, sequences, width)
        self.caches = [Kv4Cache(pool, tables[i], torch.zeros(sequences, dtype=torch.int32, device=device)) for i in range(2)]
        self.weights = [torch.zeros(sequences, kv_heads, width * page, device=device) for _ in range(2)]
        self.keep, self.recent, self.first, self.longest = keep, recent, first, 0

    @property
    def cache(self):
        return self.caches[0]

    def make_room(self, tokens):
        """Cuts the cache to ``keep`` where ``tokens`` more would not fit; whether it did."""
        if tokens > self.cache.capacity - self.keep:
            raise ValueError(f"BoundedCache: {tokens} tokens at once, {self.cache.capacity - self.keep} fit behind the {self.keep} that are kept")
        if self.longest + tokens <= self.cache.capacity:
            return False
        kv4_evict(self.caches[0], self.weights[0], self.caches[1], keep=self.keep, recent=self.recent, first=self.first, weights_out=self.weights[1])
        self.caches.reverse()
        self.weights.reverse()
        self.longest = min(self.longest, self.keep)
        return True

    def step(self, q, k, v, out, counts=None):
        """``counts`` (int32 [B]): how many of the S rows stand for tokens of each sequence; all where not given."""
        self.make_room(q.shape[1])
        self.cache.lengths.add_(q.shape[1] if counts is None else counts)
        kv4_append(self.cache, k, v, counts=counts)
        fmha_fwd_kv4(q, self.cache, out, counts=counts, weights=self.weights[0], weights_in=self.weights[0])
        self.longest += q.shape[1]   # (an upper bound: the lengths themselves are on the device)
        return out


def main(argv=None):
    import torch
    parser = argparse.ArgumentParser(description="Generation of random tokens with a bounded 4-bit cache")
    for name, value in (("sequences", 16), ("heads", 32), ("kv-heads", 8), ("prompt", 2048), ("chunk", 512), ("steps", 3000), ("room", 4096), ("keep", 2048)):
        parser.add_argument("--" + name, type=int, default=value)
    a = parser.parse_args(argv)
    layer, other = (BoundedCache(a.sequences, a.kv_heads, a.room, a.keep) for _ in range(2))

    def projections(tokens):
        x = torch.randn(a.sequences, tokens, a.heads + 2 * a.kv_heads, 128, device="cuda", dtype=torch.bfloat16)
        return (*x.split([a.heads, a.kv_heads, a.kv_heads], 2), torch.empty(a.sequences, tokens, a.heads, 128, device="cuda", dtype=torch.bfloat16))

    def timed(name, calls, work):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        evictions = work()
        end.record()
        end.synchronize()
        print(f"{name}: {start.elapsed_time(end) / calls * 1e3:.1f} us each, {calls} calls, {evictions} evictions, {layer.longest} tokens held, {layer.cache.pool.numel() / 2 / 2 ** 20:.0f} MiB for up to {a.room} each")

    def run(calls, x):
        evictions = 0
        for _ in range(calls):
            evictions += layer.make_room(x[0].shape[1])
            layer.step(*x)
        return evictions

    chunks = -(-a.prompt // a.chunk)
    chunk, token = projections(a.chunk), projections(1)
    for x in (chunk, token):   # the first calls load the kernels
        other.step(*x)
    timed(f"prompt, {a.sequences} sequences, {a.chunk} tokens at a time", chunks, lambda: run(chunks, chunk))
    timed(f"generation, {a.sequences} sequences", a.steps, lambda: run(a.steps, token))


if __name__ == "__main__":
    main()
