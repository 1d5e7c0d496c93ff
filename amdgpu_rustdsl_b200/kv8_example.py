"""Serving from a paged 8-bit cache: requests come and go, their prompts and tokens share the steps, and the pages go from one to the next without the host looking.

    python -m amdgpu_rustdsl_b200.kv8_example [--sequences 32 --layers 4 --heads 32 --kv-heads 8 --prompt 1024 --tokens 128 --steps 400 --pages 1200]

runs attention layers on random projections (there is no model here) and prints what a step takes and what became of the requests.
"""
from __future__ import annotations

import argparse

from .kv8 import Kv8Cache, fmha_fwd_kv8, kv8_append, kv8_pool
from .pages import pages_cut, pages_stack, pages_take
from .rope import Rope, rope_rotate


class PagedBatch:
    """The caches of a model's layers for ``sequences`` sequences of up to ``longest`` tokens: a pool of ``pages`` pages for each layer, one table, one set of lengths and one stack of free
    pages for all of them.

    A step is ``begin`` once, ``layer`` for each layer, and ``cut`` where tokens go: drafts that were not accepted, sequences that are over."""

    def __init__(self, sequences, layers, kv_heads, pages, longest, rope=None, page=64, device="cuda"):
        import torch
        self.table = torch.full((sequences, -(-longest // page)), -1, dtype=torch.int32, device=device)
        self.lengths, self.granted = (torch.zeros(sequences, dtype=torch.int32, device=device) for _ in range(2))
        self.caches = [Kv8Cache(kv8_pool(pages, kv_heads, page, device), self.table, self.lengths) for _ in range(layers)]
        self.free, self.rope, self.positions = pages_stack(pages, device), rope, None

    def begin(self, counts, rows):
        """Room for ``counts[b]`` (int32 [B]) new tokens of each sequence, in ``rows`` rows. Which sequences got it is in ``granted`` (counts[b] or 0) when the kernels have run: the others' rows
        stand for nothing in this step, and may be asked for again."""
        import torch
        self.positions = torch.empty((counts.shape[0], rows), dtype=torch.int32, device=counts.device)
        pages_take(self.free, self.caches[0], counts, self.granted, positions=self.positions)

    def layer(self, i, q, k, v, out):
        """One layer's attention: q, k, v bf16 [B, rows, heads, 128]; q and k are turned in place."""
        if self.rope is not None:
            rope_rotate(self.rope, q, self.positions, y=k)
        kv8_append(self.caches[i], k, v, counts=self.granted)
        fmha_fwd_kv8(q, self.caches[i], out, counts=self.granted)
        return out

    def cut(self, keep):
        """Sequences of more than ``keep[b]`` (int32 [B]) tokens are cut to that many."""
        pages_cut(self.free, self.caches[0], keep)


class Requests:
    """What the host knows of the sequences' requests: a list [tokens of the prompt, tokens in all] each, which ``new()`` makes, and how far each one is.

    One that is put off for want of pages starts again, prompt and all, when another is over: at once it would take the pages that it was put off for."""

    def __init__(self, sequences, new):
        self.new, self.now = new, [new() for _ in range(sequences)]
        self.lengths, self.waits = [0] * sequences, [False] * sequences
        self.finished, self.put_off = [], 0

    def ask(self, chunk):
        """New tokens of each sequence: prompts a chunk at a time beside the others' single tokens."""
        return [0 if wait else min(chunk, r[0] - n) if n < r[0] else 1 for n, r, wait in zip(self.lengths, self.now, self.waits)]

    def step(self, granted):
        """What becomes of the sequences: whether each is cut to nothing, or None where none is."""
        self.lengths = [n + got for n, got in zip(self.lengths, granted)]
        over = [n >= r[1] for n, r in zip(self.lengths, self.now)]
        for b, done in enumerate(over):
            if done:
                self.finished.append(self.now[b])
                self.lengths[b], self.now[b] = 0, self.new()
        if any(over):
            self.waits = [False] * len(over)
            return over
        if any(granted):
            return None
        # where nobody gets any further, the longest makes room
        b = max(range(len(over)), key=self.lengths.__getitem__)
        self.lengths[b], self.waits[b] = 0, True
        self.put_off += 1
        return [x == b for x in range(len(over))]


def main(argv=None):
    import torch
    parser = argparse.ArgumentParser(description="Requests of random lengths served from a paged 8-bit cache")
    for name, value in (("sequences", 32), ("layers", 4), ("heads", 32), ("kv-heads", 8), ("prompt", 1024), ("chunk", 256), ("tokens", 128), ("steps", 400), ("pages", 1200)):
        parser.add_argument("--" + name, type=int, default=value)
    a = parser.parse_args(argv)
    B, longest = a.sequences, a.prompt + a.tokens
    if a.pages < -(-longest // 64):
        parser.error(f"{a.pages} pages are too few for one request of {longest} tokens")
    batch = PagedBatch(B, a.layers, a.kv_heads, a.pages, longest, Rope(128, scaling={"kind": "yarn", "factor": 4.0, "original": 4096}))
    g = torch.Generator().manual_seed(1)

    def new():
        prompt = int(torch.randint(1, a.prompt + 1, (1,), generator=g))
        return [prompt, prompt + int(torch.randint(1, a.tokens + 1, (1,), generator=g))]

    requests, served, waits, us = Requests(B, new), 0, 0, []
    projections = {rows: torch.randn(B, rows, a.heads + 2 * a.kv_heads, 128, device="cuda", dtype=torch.bfloat16) for rows in (1, a.chunk)}
    for step in range(a.steps):
        asked = requests.ask(a.chunk)
        rows = 1 if max(asked) == 1 else a.chunk
        qkv, out = projections[rows], torch.empty(B, rows, a.heads, 128, device="cuda", dtype=torch.bfloat16)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        counts = torch.tensor(asked, dtype=torch.int32).cuda()
        start.record()
        batch.begin(counts, rows)
        for i in range(a.layers):
            q, k, v = qkv.clone().split([a.heads, a.kv_heads, a.kv_heads], 2)   # (a model's projections would be here)
            batch.layer(i, q, k, v, out)
        end.record()
        granted = batch.granted.tolist()
        us.append((rows, start.elapsed_time(end) * 1e3 / a.layers))
        served += sum(granted)
        waits += sum(got < want for got, want in zip(granted, asked))
        over = requests.step(granted)
        if over is not None:
            batch.cut(torch.tensor([0 if x else longest for x in over], dtype=torch.int32).cuda())
    for rows in projections:
        times = sorted(t for r, t in us if r == rows)
        if times:
            print(f"{len(times)} steps of {rows} rows: {times[len(times) // 2]:.1f} us a layer (median), projections' copy included")
    print(f"{served} tokens, {len(requests.finished)} requests finished, {waits} times one waited for pages, {requests.put_off} times one was put off; {int(batch.free[0])} of {a.pages} pages free")


if __name__ == "__main__":
    main()
