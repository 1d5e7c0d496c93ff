"""The serving operators together, as a server uses them: pages, positions, rotation, append and attention over layers that share a table, against plain products in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def turned(x, positions, rope):
    """x [n, heads, 128] in 64 bits, turned by positions [n]."""
    n = rope.rotary // 2
    angle = (positions.double()[:, None] * torch.tensor(rope.frequencies, dtype=torch.float64))[:, None]
    a, b = x[..., :n].double(), x[..., n:2 * n].double()
    cos, sin = angle.cos() * rope.factor, angle.sin() * rope.factor
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * n:].double()], -1)


@pytest.mark.parametrize("page,rotary", [(16, 128), (64, 64)])
def test_requests_come_and_go(page, rotary):
    """Prompts in pieces beside single tokens, a draft that is taken back, a sequence that ends and whose pages another one gets, and one that has to wait for pages. Every output is checked
    against the values that the cache reads back, and these against the turned keys: off by the rounding to bf16 (2^-8) and to e4m3 (2^-4, or half of its smallest step of a scale that is
    at most the largest element over 224)."""
    from amdgpu_rustdsl_b200 import Rope, kv8_read
    from amdgpu_rustdsl_b200.kv8_example import PagedBatch
    B, H, HK, layers, longest = 3, 4, 2, 2, 300
    rope = Rope(rotary, scaling={"kind": "linear", "factor": 2.0})
    pages = -(-420 // page)
    batch = PagedBatch(B, layers, HK, pages, longest, rope, page=page)
    g = torch.Generator().manual_seed(3)
    keys = [[torch.zeros(0, HK, 128, dtype=torch.float64) for _ in range(B)] for _ in range(layers)]   # turned, as they should be held
    values = [[torch.zeros(0, HK, 128, dtype=torch.float64) for _ in range(B)] for _ in range(layers)]
    lengths, waited = [0] * B, 0
    # (tokens asked for, lengths to cut to afterwards)
    for asked, keep in (([100, 64, 0], None), ([1, 90, 5], None), ([1, 1, 130], None), ([4, 4, 4], [103, 157, 137]), ([1, 1, 200], None), ([1, 1, 1], [1000, 0, 1000]), ([1, 30, 100], None), ([70, 1, 1], None)):
        rows = max(asked)
        counts = torch.tensor(asked, dtype=torch.int32, device="cuda")
        batch.begin(counts, rows)
        granted = batch.granted.tolist()
        assert all(got in (0, want) for got, want in zip(granted, asked))
        waited += sum(got < want for got, want in zip(granted, asked))
        lengths = [n + got for n, got in zip(lengths, granted)]
        assert batch.lengths.tolist() == lengths
        for layer in range(layers):
            qkv = torch.randn(B, rows, H + 2 * HK, 128, generator=g).bfloat16()
            q, k, v = qkv.cuda().split([H, HK, HK], 2)
            out = torch.full((B, rows, H, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
            batch.layer(layer, q, k, v, out)
            longest_now = max(1, max(lengths))
            held_k, held_v = (torch.empty(B, longest_now, HK, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
            kv8_read(batch.caches[layer], held_k, held_v)
            for b in range(B):
                n, m = lengths[b], granted[b]
                at = torch.arange(n - m, n)
                keys[layer][b] = torch.cat([keys[layer][b][:n - m], turned(qkv[b, :m, H:H + HK], at, rope)])
                values[layer][b] = torch.cat([values[layer][b][:n - m], qkv[b, :m, H + HK:].double()])
                if n == 0:
                    continue
                kk, vv = held_k[b, :n].double().cpu(), held_v[b, :n].double().cpu()
                for want, got in ((keys[layer][b], kk), (values[layer][b], vv)):
                    room = want.abs() * (2.0 ** -8 + 2.0 ** -4 * 1.01) + want.abs().amax() / 224 * 2.0 ** -9
                    assert ((got - want).abs() <= room).all()
                rows_q = turned(qkv[b, :m, :H], at, rope).bfloat16()
                x = torch.einsum("shd,thd->hst", rows_q.double(), kk.repeat_interleave(H // HK, 1)) / math.sqrt(128)
                x = x.masked_fill(torch.arange(n) > at[:, None], -math.inf)
                p = x.softmax(-1)
                ref = torch.einsum("hst,thd->shd", p, vv.repeat_interleave(H // HK, 1))
                # queries are rounded to bf16 once on either side, which may differ in a last place: 2^-8 |q| of each element, so of the scores' sizes, e^off - 1 of the weights
                off = 2.0 ** -7 * torch.einsum("shd,thd->hst", rows_q.double().abs(), kk.abs().repeat_interleave(H // HK, 1)).amax(-1) / math.sqrt(128) / math.sqrt(128) * 6
                spread = torch.einsum("hst,thd->shd", p, vv.abs().repeat_interleave(H // HK, 1))
                assert ((out[b, :m].cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + spread * (2.0 ** -10 + 2 * off.T[..., None])).all()
            assert all((out[b, granted[b]:] == 0).all() for b in range(B))
        if keep is not None:
            batch.cut(torch.tensor(keep, dtype=torch.int32, device="cuda"))
            lengths = [min(n, x) for n, x in zip(lengths, keep)]
            for layer in range(layers):
                for b in range(B):
                    keys[layer][b], values[layer][b] = keys[layer][b][:lengths[b]], values[layer][b][:lengths[b]]
            assert batch.lengths.tolist() == lengths
        used = sum(-(-n // page) for n in lengths)
        table = batch.table.cpu()
        mine = [int(table[b, i]) for b in range(B) for i in range(-(-lengths[b] // page))]
        free = batch.free.tolist()
        assert free[0] == pages - used and sorted(mine + free[4:4 + free[0]]) == list(range(pages))
    assert waited > 0


def test_the_command_runs(capsys):
    from amdgpu_rustdsl_b200.kv8_example import main
    main(["--sequences", "5", "--layers", "2", "--heads", "8", "--kv-heads", "2", "--prompt", "100", "--chunk", "32", "--tokens", "20", "--steps", "60", "--pages", "9"])
    text = capsys.readouterr().out
    assert "requests finished" in text and "steps of 32 rows" in text


def test_the_bounded_cache_turns_by_positions_that_outlive_evictions():
    """The 4-bit cache's example with rotary positions: the same as with rows that were turned before, through an eviction."""
    from amdgpu_rustdsl_b200 import Rope, rope_rotate
    from amdgpu_rustdsl_b200.kv4_example import BoundedCache
    rope = Rope(128)
    one, two = BoundedCache(2, 2, 128, 64, recent=16, rope=rope), BoundedCache(2, 2, 128, 64, recent=16)
    g = torch.Generator(device="cuda").manual_seed(1)
    seen = 0
    for S in (60, 1, 50, 1, 30, 1):
        q, k, v = torch.randn(2, S, 8, 128, generator=g, device="cuda").bfloat16().split([4, 2, 2], 2)
        positions = (seen + torch.arange(S, device="cuda")).int().expand(2, S)
        tq, tk = q.clone(), k.clone()
        rope_rotate(rope, tq, positions, y=tk)
        a, b = (torch.empty(2, S, 4, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        one.step(q, k, v, a)
        two.step(tq, tk, v, b)
        assert torch.equal(a, b) and torch.equal(q, tq) and torch.equal(k, tk)
        seen += S
    assert one.seen.tolist() == [seen, seen] and one.longest < seen
