"""NaN in the 4-bit cache's V: the definition makes NaN of the 32 elements of the rows that see the token, and of nothing else. Log-sum-exps and attention weights do not depend on V.

Everything else is held to the tolerances that test_gpu_kv4.py derives, against the same cache with zeros in the place of the NaN blocks."""
import math

import pytest
import torch

from tests import kv4_reference as R
from tests.test_gpu_kv4 import make_cache, no_wait_ran_out, queries  # noqa: F401

pytestmark = pytest.mark.gpu

BLOCK = 32


def put_v(cache, b, t, head, x):
    """Token t's V of one sequence and head becomes bf16 x [128], rounded as append does."""
    codes, scales, _ = R.encode(x.bfloat16()[None])
    c, s = R.record(cache.pool, int(cache.table[b, t // cache.page]), head, 1)
    c[t % cache.page], s[t % cache.page] = codes[0].cuda(), scales[0].cuda()


def caches(lengths, HK, page, spots, seed):
    """The cache with NaN in the blocks `spots` (sequence, head, token, block, size of the token's other blocks) and the one with zeros there."""
    both = [make_cache(lengths, HK, page, seed=seed) for _ in range(2)]
    g = torch.Generator().manual_seed(seed + 1)
    for b, head, t, block, size in spots:
        x = torch.randn(128, generator=g) * size
        for cache, what in zip(both, (math.inf, 0.0)):
            y = x.clone()
            y[BLOCK * block:BLOCK * (block + 1)] = 0.0
            y[BLOCK * block + 5] = what
            put_v(cache, b, t, head, y)
    return both


def check(lengths, HK, group, S, page, spots, causal, counts=None, seed=51):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    dirty, clean = caches(lengths, HK, page, spots, seed)
    B, H = len(lengths), HK * group
    q = queries(B, S, H)
    out, lse = torch.full((B, S, H, 128), -5.0, dtype=torch.bfloat16, device="cuda"), torch.full((B, H, S), -5.0, device="cuda")
    weights = torch.full((B, HK, dirty.capacity), -7.0, device="cuda")
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    fmha_fwd_kv4(q, dirty, out, causal=causal, counts=n, lse=lse, weights=weights)
    ref, ref_lse, ref_w, spread, peak, size, doubt = R.attend(q.cpu(), clean.pool.cpu(), clean.table.cpu(), clean.lengths.cpu(), causal, counts)
    nan = torch.zeros(ref.shape, dtype=torch.bool)
    for b, head, t, block, _ in spots:
        rows = min(S, lengths[b]) if counts is None else min(S, lengths[b], counts[b])
        for i in range(rows):
            if not causal or t <= lengths[b] - rows + i:
                nan[b, i, head * group:(head + 1) * group, BLOCK * block:BLOCK * (block + 1)] = True
    got = out.cpu().double()
    assert torch.equal(torch.isnan(got), nan), (int(torch.isnan(got).sum()), int(nan.sum()))
    off = 128 * 2.0 ** -24 * size + 2.0 ** -21
    room = 2.0 ** -9 * ref.abs() + spread * (2.0 ** -9 + 4 * off.permute(0, 2, 1)[..., None]) * 1.01 + (max(lengths) * 1.5 * 2.0 ** -25 * peak)[..., None] + 1e-38
    assert ((got - ref).abs() <= room)[~nan].all(), ((got - ref).abs() / room)[~nan].max()
    lse, some = lse.cpu().double(), ref_lse != -math.inf
    assert torch.equal(lse == -math.inf, ~some)
    assert ((lse - ref_lse).abs() <= off + 2.0 ** -22 * ref_lse.abs())[some].all()
    live = (torch.arange(dirty.capacity) < dirty.lengths.cpu()[:, None, None]).expand_as(ref_w)
    w = weights.cpu().double()
    assert ((w - ref_w).abs() <= 2 * (128 * 2.0 ** -24 * doubt + 2.0 ** -20 * ref_w.abs()) + 1e-30)[live].all() and (w[~live] == -7.0).all()


# rows of a KV head: 4, 12, 20 and 32 are the groups of eight of the decode kernel, more go to the tensor cores' tiles
SHAPES = [(1, 4, 16), (3, 4, 32), (5, 4, 64), (8, 4, 16), (9, 4, 64), (40, 4, 32), (130, 2, 128), (300, 1, 16)]


@pytest.mark.parametrize("S,group,page", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_a_block_of_a_token(S, group, page, causal):
    """The last token, one in the middle, the first, and two blocks of one token; heads without NaN beside them."""
    check([260, 90, 50], 2, group, S, page, [(0, 0, 259, 1, 1.0), (0, 0, 100, 3, 1.0), (1, 1, 0, 0, 1.0), (2, 0, 30, 2, 1.0)], causal)


@pytest.mark.parametrize("S,group", [(1, 4), (6, 4), (40, 4), (257, 2)])
def test_where_items_are_cut_between_ctas(S, group):
    """A long sequence whose partial results are put together, rows that stand for nothing beside it."""
    check([3001, 600], 1, group, S, 64, [(0, 0, 1500, 1, 1.0), (0, 0, 2998, 2, 1.0), (1, 0, 599, 0, 1.0)], True, counts=[S, min(S, 3)])


@pytest.mark.parametrize("S,group,page", SHAPES)
def test_the_blocks_beside_it_may_be_larger_than_everything_around(S, group, page):
    """What is left of the token counts with its own scales: alone among 32 and 128 tokens, and 2^20 times what the tokens beside it hold."""
    check([129, 33, 200], 2, group, S, page, [(0, 0, 128, 2, 1.0), (1, 1, 32, 0, 1.0), (2, 0, 77, 1, 2.0 ** 20), (2, 1, 199, 3, 2.0 ** 20)], True)


@pytest.mark.parametrize("S", [1, 5, 40])
def test_a_weight_too_small_for_16_bits_still_meets_nan(S):
    """One key has all the weight; the token with NaN, four behind it among the last, partly masked tokens, is seen with a weight far below 2^-25."""
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    cache = make_cache([40], 1, 16, seed=61)
    q = queries(1, S, 1, gain=0.0)
    q[0] = q[0, 0]
    codes, scales, _ = R.encode((q[0, 0, 0].float() * 32).bfloat16().cpu()[None])
    c, s = R.record(cache.pool, int(cache.table[0, 2]), 0, 0)
    c[1], s[1] = codes[0].cuda(), scales[0].cuda()
    x = torch.randn(128, generator=torch.Generator().manual_seed(3))
    x[40] = math.nan
    put_v(cache, 0, 37, 0, x)
    k, _ = R.tokens(cache.pool.cpu(), cache.table[0].tolist(), 0, 40)
    score = k @ q[0, 0, 0].cpu().double() / math.sqrt(128)
    assert score[37] - score[33] < -40   # (e^-40 < 2^-57)
    out = torch.empty_like(q)
    fmha_fwd_kv4(q, cache, out)
    for i in range(S):
        bad = torch.isnan(out[0, i, 0]).cpu()
        expect = torch.zeros(128, dtype=torch.bool)
        expect[32:64] = 40 - S + i >= 37
        assert torch.equal(bad, expect), i
