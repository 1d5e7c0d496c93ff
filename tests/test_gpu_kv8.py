"""The operators around the 8-bit cache on the GPU, against their definition in 64 bits (kv8_reference.py).

Tolerances. A score is a sum of 128 exact products in f32, whose additions may be cut off in place of rounded: off by 128 * 2^-23 of the sum of their sizes, `size` per row, by 2^-21
of itself at most through the factors and by 2^-21 through exp2 or log2: `off`, what a log-sum-exp may be off (with its own rounding). A weight p is off by 2 `off` relative, its own and
the sum's, so that an output is off by 4 `off` of sum p |v|, by 2^-11 of that since weights go into the second product in f16, by 2^-8 of itself as bf16, and where weights come out subnormal
in f16 by 2^-25 * 448 for each token, against a largest weight times V's scale, `peak`, of 2^6 or more. What is held in 8 bits is equal."""
import math

import pytest
import torch

from tests import kv8_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    """No kernel gave up a wait (the status word is the process's: earlier tests' kernels count too)."""
    from amdgpu_rustdsl_b200 import device_status
    before = device_status()
    yield
    assert device_status() == before


def fill(lengths, HK, page, seed=0, width=None, extra=3, k_gain=None, v_gain=None, garbage=0xFF):
    """pool, table, lengths on the CPU: normal keys and values; pages in random order; unused pages and what is behind the lengths hold `garbage` bytes (0xFF: NaN codes and scales)."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    width = max(1, max(counts)) if width is None else width
    total = sum(counts) + extra
    pool = torch.full((total, HK, 257 * page), garbage, dtype=torch.uint8)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    order = torch.randperm(total, generator=g).tolist()
    for b, n in enumerate(counts):
        for i in range(n):
            table[b, i] = order.pop()
    S = max(lengths)
    if S:
        k, v = (torch.zeros(len(lengths), S, HK, 128) for _ in range(2))
        for b, n in enumerate(lengths):
            for x, gain in ((k, k_gain), (v, v_gain)):
                y = torch.randn(n, HK, 128, generator=g)
                x[b, :n] = y if gain is None else y * gain(g, n)[:, None]
        R.append(pool, table, lengths, lengths, k.bfloat16(), v.bfloat16())
    return pool, table, torch.tensor(lengths, dtype=torch.int32)


def make_cache(lengths, HK, page, **how):
    from amdgpu_rustdsl_b200 import Kv8Cache
    return Kv8Cache(*(x.cuda() for x in fill(lengths, HK, page, **how)))


def queries(B, S, H, seed=1, gain=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, S, H, 128, generator=g) * torch.exp2(torch.rand(H, 1, generator=g) * gain - 1)).bfloat16().cuda()


def room_of(ref, spread, peak, size, lse, tokens):
    """What outputs and log-sum-exps may be off (lse: [B, H, S])."""
    off = 130 * 2.0 ** -23 * size + 2.0 ** -20
    each = lambda x: x.permute(0, 2, 1)[..., None]
    return 2.0 ** -8 * ref.abs() + spread * (2.0 ** -11 + 4 * each(off)) + tokens * 2.0 ** -31 * 448 * each(peak) + 1e-38, off + 2.0 ** -22 * lse.abs()


def check_attend(cache, q, causal=True, counts=None, scale=None, **call):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv8
    B, S, H, _ = q.shape
    out = torch.full((B, S, H, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    lse = torch.full((B, H, S), float("nan"), device="cuda")
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    fmha_fwd_kv8(q, cache, out, causal=causal, counts=n, scale=scale, lse=lse, **call)
    again = torch.full_like(out, float("nan"))
    fmha_fwd_kv8(q, cache, again, causal=causal, counts=n, scale=scale, **call)
    torch.cuda.synchronize()
    ref, ref_lse, spread, peak, size = R.attend(q.cpu(), cache.pool.cpu(), cache.table.cpu(), cache.lengths.tolist(), causal, counts, scale)
    assert torch.equal(out, again)
    got, lse = out.cpu().double(), lse.cpu().double()
    assert torch.isfinite(got).all()
    none = ref_lse == -math.inf
    room, lse_room = room_of(ref, spread, peak, size, ref_lse.masked_fill(none, 0.0), max(1, int(cache.lengths.max())))
    assert ((got - ref).abs() <= room).all(), ((got - ref).abs() / room).max()
    assert torch.equal(lse == -math.inf, none)
    assert ((lse - ref_lse).abs()[~none] <= lse_room[~none]).all()
    return out


SHAPES = [
    # lengths, HK, group, S, page
    ([1], 1, 1, 1, 16), ([2, 0, 1], 2, 4, 1, 16), ([15, 16, 17], 1, 8, 1, 16), ([31, 32, 33, 63, 64, 65], 2, 4, 1, 32), ([127, 128, 129], 2, 3, 1, 64), ([255, 257, 5], 1, 16, 1, 128),
    ([1000, 1, 0, 333], 2, 5, 1, 64), ([700], 1, 2, 1, 128), ([129, 48], 2, 12, 1, 16), ([300, 77], 2, 4, 2, 64), ([300, 3], 1, 4, 5, 32), ([511, 130], 2, 8, 3, 64), ([90], 1, 16, 2, 16),
    ([260, 33], 1, 4, 33, 64), ([140, 9], 1, 8, 40, 32), ([131], 2, 1, 131, 16), ([257, 64, 0], 1, 3, 64, 128), ([200], 1, 16, 17, 64), ([385, 129], 2, 7, 60, 64), ([530, 17], 1, 2, 300, 16),
]


@pytest.mark.parametrize("lengths,HK,group,S,page", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_attention(lengths, HK, group, S, page, causal):
    cache = make_cache(lengths, HK, page, seed=sum(lengths))
    check_attend(cache, queries(len(lengths), S, HK * group), causal)


def test_rows_that_stand_for_nothing():
    """counts between nothing and all rows, cut where they exceed the rows or the length, below 0 none."""
    cache = make_cache([100, 40, 3, 70, 0], 2, 32)
    check_attend(cache, queries(5, 6, 8), True, counts=[0, 4, 5, -3, 2])
    check_attend(cache, queries(5, 6, 8), False, counts=[6, 100, 1, 2, 0])
    check_attend(cache, queries(5, 50, 8), True, counts=[7, 40, 3, 50, 1])


@pytest.mark.parametrize("S", [1, 40])
def test_lengths_beyond_the_table_are_cut(S):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv8
    cache = make_cache([64, 64], 1, 16)
    cache.lengths.copy_(torch.tensor([1000, -5], dtype=torch.int32))
    q = queries(2, S, 4)
    out, same = torch.full_like(q, float("nan")), torch.full_like(q, float("nan"))
    fmha_fwd_kv8(q, cache, out)
    cache.lengths.copy_(torch.tensor([64, 0], dtype=torch.int32))
    fmha_fwd_kv8(q, cache, same)
    assert torch.equal(out, same) and (out[1] == 0).all() and torch.isfinite(out).all()


@pytest.mark.parametrize("S", [1, 40])
def test_a_wider_table_changes_nothing_behind_the_length(S):
    lengths = [130, 50]
    a, b = make_cache(lengths, 2, 32, seed=3), make_cache(lengths, 2, 32, seed=3, width=200)
    b.table[:, 5:] = 0x7FFFFFFF
    q = queries(2, S, 8)
    check_attend(a, q)
    check_attend(b, q)


@pytest.mark.parametrize("S,group", [(1, 4), (3, 8), (48, 4)])
def test_scales_of_v_from_tiny_to_huge(S, group):
    """Tokens whose values differ by many binades, within a block and between blocks, blocks of zeros among them."""
    def gain(g, n):
        block = torch.exp2(torch.randint(-30, 30, (-(-n // 16), 1), generator=g).float()) * (torch.rand(-(-n // 16), 1, generator=g) > 0.1)
        return block.repeat_interleave(16, 0)[:n] * torch.exp2(torch.randint(-6, 6, (n, 1), generator=g).float())
    check_attend(make_cache([150, 70], 1, 16, seed=5, v_gain=gain), queries(2, S, group))


@pytest.mark.parametrize("v_exponent", [-126, -70, 60, 100, 120])
@pytest.mark.parametrize("S", [1, 36])
def test_values_at_the_ends_of_the_range(S, v_exponent):
    cache = make_cache([90], 1, 32, seed=6, v_gain=lambda g, n: torch.full((n, 1), 2.0 ** v_exponent))
    check_attend(cache, queries(1, S, 4))


@pytest.mark.parametrize("k_exponent,q_exponent", [(90, 0), (90, -90), (-85, 0), (-85, 60), (-60, 100), (0, 100), (0, -90), (20, 100), (98, 20)])
@pytest.mark.parametrize("S", [1, 6, 40])
def test_keys_and_queries_of_any_size(S, k_exponent, q_exponent):
    """The scale brings the scores back to the ordinary."""
    cache = make_cache([150, 33], 1, 16, seed=95, k_gain=lambda g, n: torch.full((n, 1), 2.0 ** k_exponent))
    check_attend(cache, queries(2, S, 4) * 2.0 ** q_exponent, scale=2.0 ** -(k_exponent + q_exponent) / math.sqrt(128))


@pytest.mark.parametrize("S", [1, 6, 40])
def test_keys_of_many_sizes_in_one_sequence(S):
    def gain(g, n):
        return torch.exp2(torch.randint(-12, 2, (n, 1), generator=g).float())
    check_attend(make_cache([400, 129], 2, 64, seed=96, k_gain=gain), queries(2, S, 8))


@pytest.mark.parametrize("S", [1, 34])
def test_rows_that_grow_late(S):
    """Scores that rise along the sequence, so that the running reference moves again and again."""
    def gain(g, n):
        return torch.linspace(0.1, 6, n)[:, None]
    check_attend(make_cache([400], 1, 64, seed=7, k_gain=gain), queries(1, S, 4, gain=3.0))


@pytest.mark.parametrize("S", [1, 40])
def test_other_scales_and_zero_queries(S):
    cache = make_cache([200, 33], 2, 64, seed=9)
    q = queries(2, S, 8)
    check_attend(cache, q, scale=0.5)
    check_attend(cache, q, scale=1e-3)
    q[0] = 0
    q[1, :, 3] *= 2.0 ** -100
    check_attend(cache, q)


def spoil(cache, b, t, part, head=0):
    """Token t of a sequence holds no numbers in K (part 0) or V, as append leaves it."""
    pool = cache.pool.cpu()
    block = R.block_at(pool, cache.table.cpu(), b, head, t)
    block.set_codes(part, torch.tensor([t % 16]), torch.zeros(1, 128, dtype=torch.uint8))
    block.set_meta(part, block.scale(part), block.mask(part) | 1 << t % 16)
    cache.pool.copy_(pool)


@pytest.mark.parametrize("rows,group", [(2, 4), (5, 4), (40, 4), (300, 1)])
@pytest.mark.parametrize("part", [0, 1])
def test_tokens_without_numbers_reach_the_rows_that_see_them(rows, group, part):
    """The last token is seen by the last row alone, one in the middle of the new ones by half of them; a token with a vanishing weight counts too. Other rows are as they were."""
    from amdgpu_rustdsl_b200 import fmha_fwd_kv8
    for t in (399, 399 - rows // 2, 400 - rows):
        cache = make_cache([400, 33], 1, 32, seed=10)
        q = queries(2, rows, group)
        good, good_lse = torch.empty_like(q), torch.empty(2, group, rows, device="cuda")
        fmha_fwd_kv8(q, cache, good, lse=good_lse)
        spoil(cache, 0, t, part)
        out, lse = torch.empty_like(q), torch.empty_like(good_lse)
        fmha_fwd_kv8(q, cache, out, lse=lse)
        first = t - (400 - rows)   # the first row that sees it
        assert torch.isnan(out[0, first:]).all() and torch.equal(out[0, :first], good[0, :first]) and torch.equal(out[1], good[1])
        if part == 0:
            assert torch.isnan(lse[0, :, first:]).all() and torch.equal(lse[0, :, :first], good_lse[0, :, :first])
        else:   # its code is 0 and its scale as it was
            assert torch.equal(lse, good_lse)
        everyone = torch.empty_like(q)
        fmha_fwd_kv8(q, cache, everyone, causal=False)
        assert torch.isnan(everyone[0]).all() and torch.isfinite(everyone[1, :33]).all()


@pytest.mark.parametrize("S", [1, 40])
def test_infinite_and_nan_queries_stay_in_their_rows(S):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv8
    cache = make_cache([100], 1, 32, seed=11)
    q = queries(1, S, 4)
    good = torch.empty_like(q)
    fmha_fwd_kv8(q, cache, good)
    bad = q.clone()
    bad[0, 0, 1, 5] = float("nan")
    bad[0, 0, 2, 7] = float("inf")
    out = torch.empty_like(q)
    fmha_fwd_kv8(bad, cache, out)
    assert torch.isnan(out[0, 0, 1]).all() and torch.isnan(out[0, 0, 2]).any()
    keep = torch.ones(S, 4, dtype=torch.bool)
    keep[0, 1:3] = False
    assert torch.equal(out[0][keep.cuda()], good[0][keep.cuda()])


@pytest.mark.parametrize("S", [1, 5, 40])
@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31])
@pytest.mark.parametrize("page", [16, 32])
def test_pages_outside_the_pool_are_never_followed(S, bad, page):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv8
    cache = make_cache([100, 100], 1, page, seed=12)
    q = queries(2, S, 4)
    good = torch.empty_like(q)
    fmha_fwd_kv8(q, cache, good)
    cache.table[0, 1] = bad
    out = torch.empty_like(q)
    fmha_fwd_kv8(q, cache, out)
    assert torch.isnan(out[0]).all() and torch.equal(out[1], good[1])   # every row sees the second page


@pytest.mark.parametrize("S", [1, 40])
def test_strided_queries_other_streams_and_graphs(S):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv8
    cache = make_cache([200, 90], 2, 64, seed=14)
    wide = torch.zeros(2, S, 3, 8, 128, dtype=torch.bfloat16, device="cuda")
    q = queries(2, S, 8)
    wide[:, :, 1] = q
    good = check_attend(cache, q)
    assert torch.equal(check_attend(cache, wide[:, :, 1]), good)
    stacked = q.transpose(1, 2).contiguous().transpose(1, 2)   # [B, H, S, 128] in memory
    assert torch.equal(check_attend(cache, stacked), good)
    within = q.clone()
    fmha_fwd_kv8(within, cache, within)
    assert torch.equal(within, good)
    side = torch.cuda.Stream()
    late = torch.zeros_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)   # the queries arrive on the side stream only after a while
        late.copy_(q)
        out = torch.empty_like(q)
        fmha_fwd_kv8(late, cache, out)
    side.synchronize()
    assert torch.equal(out, good)
    out.zero_()
    torch.cuda.synchronize()
    fmha_fwd_kv8(q, cache, out, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, good)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = [torch.empty_like(q) for _ in graphs]
    with torch.cuda.stream(side):
        fmha_fwd_kv8(q, cache, out)
    side.synchronize()
    for graph, o in zip(graphs, outs):
        with torch.cuda.graph(graph, stream=side):
            fmha_fwd_kv8(q, cache, o)
    for n in (200, 137):
        cache.lengths[0] = n
        good = check_attend(cache, q)
        torch.cuda.synchronize()
        other = torch.cuda.Stream()
        for graph, o, s in zip(graphs, outs, (side, other)):   # two replays at once
            o.zero_()
            torch.cuda.synchronize()
        for graph, s in zip(graphs, (side, other)):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, good) for o in outs)


def test_a_pool_beyond_32_bits():
    """Pages more than 2^32 bytes apart."""
    from amdgpu_rustdsl_b200 import Kv8Cache, fmha_fwd_kv8, kv8_append, kv8_read
    page, HK = 128, 8
    pages = (5 << 30) // (HK * 257 * page)
    pool = torch.empty(pages, HK, 257 * page, dtype=torch.uint8, device="cuda")
    table = torch.tensor([[pages - 1, 0], [3, pages - 2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([200, 256], dtype=torch.int32, device="cuda")
    big = Kv8Cache(pool, table, lengths)
    small = Kv8Cache(torch.empty(4, HK, 257 * page, dtype=torch.uint8, device="cuda"), torch.tensor([[2, 0], [3, 1]], dtype=torch.int32, device="cuda"), lengths)
    g = torch.Generator(device="cuda").manual_seed(4)
    k, v = (torch.randn(2, 256, HK, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
    counts = torch.tensor([200, 256], dtype=torch.int32, device="cuda")
    got = []
    for cache in (big, small):
        kv8_append(cache, k, v, counts=counts)
        rk, rv = torch.empty_like(k), torch.empty_like(v)
        kv8_read(cache, rk, rv)
        out = []
        for S in (1, 40):
            q = queries(2, S, 32)
            out.append(torch.empty_like(q))
            fmha_fwd_kv8(q, cache, out[-1])
        got.append([rk, rv] + out)
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("B,HK,H,L,S", [(1, 1, 4, 70001, 1), (3, 2, 16, 20011, 1), (1, 2, 8, 30003, 5), (1, 1, 8, 5000, 700), (2, 2, 2, 3001, 1500), (150, 8, 32, 100, 1), (2, 1, 12, 9001, 2)])
def test_many_tiles_against_a_plain_product(B, HK, H, L, S):
    """Long sequences, cut between many CTAs, against the same sums in f64 on the GPU."""
    from amdgpu_rustdsl_b200 import Kv8Cache, fmha_fwd_kv8, kv8_append, kv8_pool, kv8_read
    per = -(-L // 64)
    cache = Kv8Cache(kv8_pool(B * per, HK), torch.randperm(B * per, device="cuda").int().view(B, per), torch.full((B,), L, dtype=torch.int32, device="cuda"))
    g = torch.Generator(device="cuda").manual_seed(L)
    k, v = (torch.randn(B, L, HK, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
    kv8_append(cache, k, v)
    kv8_read(cache, k, v)
    q = (torch.randn(B, S, H, 128, generator=g, device="cuda") * 2).bfloat16()
    out, lse = torch.empty_like(q), torch.empty(B, H, S, device="cuda")
    fmha_fwd_kv8(q, cache, out, lse=lse)
    at = torch.arange(L - S, L, device="cuda")
    for b in {0, B - 1}:
        for hk in {0, HK - 1}:
            kk, vv = k[b, :, hk].double(), v[b, :, hk].double()
            for h in range(hk * (H // HK), (hk + 1) * (H // HK)):
                rows, hidden = q[b, :, h].double(), torch.arange(L, device="cuda") > at[:, None]
                x = (rows @ kk.T / math.sqrt(128)).masked_fill_(hidden, -math.inf)
                ref_lse = torch.logsumexp(x, 1)
                p = torch.exp(x - ref_lse[:, None])
                ref, spread = p @ vv, p @ vv.abs()
                # V's scales are 2^-5 at most (values below 8), a row's largest weight times that
                peak = p.amax(1) * 2.0 ** -5
                size = (rows.abs() @ kk.abs().T / math.sqrt(128)).amax(1)
                room, lse_room = room_of(ref[None, :, None], spread[None, :, None], peak[None, None], size[None, None], ref_lse[None, None], L)
                assert ((out[b, :, h].double() - ref).abs() <= room[0, :, 0]).all()
                assert ((lse[b, h].double() - ref_lse).abs() <= lse_room[0, 0]).all()


def test_back_to_back_calls_give_the_same():
    """Many launches without a wait between them, of work that is cut between CTAs in the middle of items: none stalls, all give the same bits."""
    from amdgpu_rustdsl_b200 import fmha_fwd_kv8
    cache = make_cache([3000, 1500], 2, 64, seed=15)
    for S in (1, 4, 100, 300):
        q = queries(2, S, 8)
        first, out = torch.empty_like(q), torch.empty_like(q)
        fmha_fwd_kv8(q, cache, first)
        for _ in range(200):
            fmha_fwd_kv8(q, cache, out)
        torch.cuda.synchronize()
        assert torch.equal(out, first)


# ------------------------------------------------------------------------------------------------- append and read
def same_values(got, want):
    """Equal, NaN at the same places, zeros of the same sign."""
    got, want = got.cpu(), want.cpu()
    return torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(0), want.nan_to_num(0)) and torch.equal(torch.signbit(got)[~torch.isnan(got)], torch.signbit(want)[~torch.isnan(want)])


def check_append(cache, k, v, counts=None):
    """Every byte of the pool that belongs to a sequence's tokens, scales and masks is as the definition says, and nothing else has changed."""
    from amdgpu_rustdsl_b200 import kv8_append, kv8_read
    expect, table, lengths = cache.pool.cpu().clone(), cache.table.cpu(), cache.lengths.tolist()
    R.append(expect, table, lengths, counts, k.cpu(), v.cpu())
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    kv8_append(cache, k, v, counts=n)
    got = cache.pool.cpu()
    # the place behind an odd last token may be written: it holds nothing
    new = R.new_tokens(lengths, counts, k.shape[1])
    for b, (L, m) in enumerate(zip(lengths, new)):
        if m and L % 2 and R.block_at(got, table, b, 0, L - 1) is not None:
            for h in range(got.shape[1]):
                R.block_at(expect, table, b, h, L - 1).set_codes(1, torch.tensor([L % 16]), R.block_at(got, table, b, h, L - 1).codes(1)[L % 16][None])
    assert torch.equal(got, expect)
    held = [torch.full(k.shape, 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    kv8_read(cache, held[0], held[1], last=True, counts=n)
    for b, (L, m) in enumerate(zip(lengths, new)):
        for h in range(k.shape[2]):
            values = R.tokens(expect, table, b, h, L)[:2]
            for part in (0, 1):
                assert same_values(held[part][b, :m, h], values[part][L - m:].bfloat16())
        assert (held[0][b, m:] == 0).all() and (held[1][b, m:] == 0).all()


def test_append_rounds_every_bf16_value_as_the_definition_does():
    """All 65536 bf16 bit patterns among others, and finite ones as the largest of their block; whole blocks of zeros; Inf and NaN."""
    from amdgpu_rustdsl_b200 import Kv8Cache
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    g = torch.Generator().manual_seed(3)
    rows = [bits.view(-1, 128), bits[torch.randperm(65536, generator=g)].view(-1, 128)]
    finite = bits[torch.isfinite(bits.float())]
    top = finite[torch.randperm(len(finite), generator=g)[:160]]   # one a block
    near = (top[:, None].float() * torch.rand(160, 16 * 128, generator=g) * torch.exp2(-torch.randint(0, 20, (160, 16 * 128), generator=g).float()))
    near[:, 77] = top.float()
    rows.append(near.bfloat16().view(-1, 128))
    rows.append(torch.zeros(32, 128).bfloat16())
    x = torch.cat(rows)
    n = len(x) // 2
    for page in (16, 64):
        width = -(-n // page)
        cache = Kv8Cache(torch.full((width, 1, 257 * page), 0x77, dtype=torch.uint8, device="cuda"), torch.randperm(width, generator=g).int()[None].cuda(), torch.tensor([n], dtype=torch.int32).cuda())
        check_append(cache, x[:n].view(1, n, 1, 128).cuda(), x[n:2 * n].view(1, n, 1, 128).cuda())


@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_writes_its_tokens_and_nothing_else(page):
    """Ragged numbers of new tokens from strided rows, over ends of blocks and pages, onto bytes that must stay; a page outside the pool drops its tokens."""
    lengths, counts, S, HK = [130, 1, 0, 70, 33, 200, 37], [9, 1, 3, 0, 40, -1, 4], 9, 3
    cache = make_cache(lengths, HK, page, seed=21, garbage=0x5A)
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(7, S, 4 + 2 * HK, 128, generator=g).bfloat16().cuda()
    k, v = qkv[:, :, 4:4 + HK], qkv[:, :, 4 + HK:]
    lost = int(cache.table[0, 129 // page])
    cache.table[0, 129 // page] = 10 ** 6
    check_append(cache, k, v, counts)
    cache.table[0, 129 // page] = lost
    check_append(cache, k, v)   # without counts: as many as there are, up to the length


@pytest.mark.parametrize("steps", [[1] * 40, [3] * 12, [17, 1, 15, 2, 31], [5, 11, 16, 1]])
def test_scales_that_grow_as_tokens_come(steps):
    """Tokens of a block come in several calls, larger and smaller ones, with NaN and Inf here and there: older codes follow the scale, masks stay, blocks of one part do not notice the other."""
    cache = make_cache([0, 5], 2, 32, seed=22, width=4)
    cache.table.copy_(torch.arange(8).view(2, 4).flip(0).int())
    cache = type(cache)(torch.full((8, 2, 257 * 32), 0xFF, dtype=torch.uint8, device="cuda"), cache.table, cache.lengths)
    cache.lengths.zero_()
    g = torch.Generator().manual_seed(sum(steps))
    for n in steps:
        k, v = (torch.randn(2, n, 2, 128, generator=g) * torch.exp2(torch.randint(-14, 15, (2, n, 2, 1), generator=g).float()) for _ in range(2))
        for x in (k, v):
            x[torch.rand(2, n, 2, 128, generator=g) < 0.0005] = math.inf
            x[torch.rand(2, n, 2, 128, generator=g) < 0.0005] = math.nan
        cache.lengths += n
        check_append(cache, k.bfloat16().cuda(), v.bfloat16().cuda())


def test_tokens_that_are_taken_back_and_written_again():
    """Lengths go down and up again: what is written depends on what is held in front alone, and on the block's scale."""
    cache = make_cache([45, 20], 1, 16, seed=23)
    g = torch.Generator().manual_seed(9)
    for lengths, n in (([40, 16], 3), ([48, 32], 7), ([41, 17], 1), ([47, 31], 15)):
        cache.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        check_append(cache, *((torch.randn(2, n, 1, 128, generator=g) * 2.0 ** int(torch.randint(-3, 4, (1,), generator=g))).bfloat16().cuda() for _ in range(2)))


def test_read_from_the_start_and_into_strided_rows():
    from amdgpu_rustdsl_b200 import kv8_read
    lengths = [70, 0, 5]
    cache = make_cache(lengths, 2, 32, seed=22)
    wide = torch.full((3, 80, 5, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    kv8_read(cache, wide[:, :, 0:2], wide[:, :, 3:5])
    assert (wide[:, :, 2] == 9).all()
    for b, n in enumerate(lengths):
        for h in range(2):
            k, v, _ = R.tokens(cache.pool.cpu(), cache.table.cpu(), b, h, n)
            assert torch.equal(wide[b, :n, h].cpu().double(), k) and torch.equal(wide[b, :n, 3 + h].cpu().double(), v)
        assert (wide[b, n:, :2] == 0).all() and (wide[b, n:, 3:] == 0).all()


def test_refusals_of_the_python_entry():
    from amdgpu_rustdsl_b200 import Kv4Cache, fmha_fwd_kv8, kv4_pool, kv8_append, kv8_read
    cache = make_cache([40, 20], 2, 16, seed=41)
    q = queries(2, 1, 8)
    out = torch.empty_like(q)
    for bad, message in ((q.float(), "bf16"), (q[..., :64], "bf16"), (q[:1], "bf16"), (q.cpu(), "device"), (q.transpose(2, 3).contiguous().transpose(2, 3), "dense")):
        with pytest.raises(ValueError, match=message):
            fmha_fwd_kv8(bad, cache, out)
    odd = torch.empty(2 * 8 * 128 + 8, dtype=torch.bfloat16, device="cuda")[4:-4].view(2, 1, 8, 128)
    with pytest.raises(ValueError, match="16 bytes"):
        fmha_fwd_kv8(odd, cache, out)
    for bad in (out.float(), out[:, :, :4]):
        with pytest.raises(ValueError):
            fmha_fwd_kv8(q, cache, bad)
    for heads in (34, 3):
        with pytest.raises(ValueError, match="1 to 16 times"):
            fmha_fwd_kv8(queries(2, 1, heads), cache, torch.empty(2, 1, heads, 128, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError, match="counts"):
        fmha_fwd_kv8(q, cache, out, counts=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="lse"):
        fmha_fwd_kv8(q, cache, out, lse=torch.empty(2, 1, 8, device="cuda"))
    with pytest.raises(ValueError, match="scale"):
        fmha_fwd_kv8(q, cache, out, scale=-1.0)
    wide = torch.zeros(2, 1, 16, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="packed"):
        fmha_fwd_kv8(wide[:, :, ::2], cache, wide.view(-1)[:2 * 8 * 128].view(2, 1, 8, 128))
    k = torch.empty(2, 3, 2, 128, dtype=torch.bfloat16, device="cuda")
    for args in ((k, k[:, :2]), (k[:, :, :1], k), (k.half(), k)):
        with pytest.raises(ValueError):
            kv8_append(cache, *args)
        with pytest.raises(ValueError):
            kv8_read(cache, *args)
    with pytest.raises(ValueError, match="counts"):
        kv8_read(cache, k, k, counts=cache.lengths)
    other = Kv4Cache(kv4_pool(4, 2, 16), cache.table, cache.lengths)
    for call in (lambda: kv8_append(other, k, k), lambda: kv8_read(other, k, k), lambda: fmha_fwd_kv8(q, other, out)):
        with pytest.raises(ValueError, match="Kv8Cache"):
            call()
