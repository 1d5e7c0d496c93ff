"""The operators around the 4-bit cache on the GPU, against their definition in 64 bits (kv4_reference.py).

Tolerances. A score is a sum of 128 exact products in f32: off by at most 128 * 2^-24 of the sum of their sizes, `size` per row; with exp2 and log2 (2^-21 here) this
is what the log-sum-exps and, doubled and times the weight, the attention weights may be off. An output is rounded to bf16 (2^-9 of itself); the weights that
multiply V are rounded to f16 or bf16 (2^-9 of sum p |v| at most), and in f16 those below 2^-24 of the row's largest product vanish (1.5 * 2^-25 of it per token:
a block's largest code is 4 or 6). What is held in 4 bits, positions and lengths are equal."""
import math

import pytest
import torch

from tests import kv4_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    """No kernel gave up a wait (the status word is the process's: earlier tests' kernels count too)."""
    from amdgpu_rustdsl_b200 import device_status
    before = device_status()
    yield
    assert device_status() == before


def make_cache(lengths, HK, page, seed=0, width=None, extra=3, k_gain=None, v_gain=None, garbage=0xFF):
    """A cache with normal keys and values; pages in random order; unused pages and tokens behind the lengths hold `garbage` bytes (0xFF: NaN scales)."""
    from amdgpu_rustdsl_b200 import Kv4Cache
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    width = max(1, max(counts)) if width is None else width
    total = sum(counts) + extra
    pool = torch.full((total, HK, 136 * page), garbage, dtype=torch.uint8)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    order = torch.randperm(total, generator=g).tolist()
    for b, n in enumerate(counts):
        for i in range(n):
            table[b, i] = order.pop()
    for b, n in enumerate(lengths):
        for h in range(HK):
            for part, gain in ((0, k_gain), (1, v_gain)):
                x = torch.randn(n, 128, generator=g)
                x = x if gain is None else x * gain(g, n)
                codes, scales, _ = R.encode(x.bfloat16())
                for i in range(-(-n // page)):
                    c, s = R.record(pool, int(table[b, i]), h, part)
                    m = min(page, n - i * page)
                    c[:m], s[:m] = codes[i * page:i * page + m], scales[i * page:i * page + m]
    return Kv4Cache(pool.cuda(), table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda())


def queries(B, S, H, seed=1, gain=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, S, H, 128, generator=g) * torch.exp2(torch.rand(H, 1, generator=g) * gain - 1)).bfloat16().cuda()


def check_attend(cache, q, causal=True, counts=None, scale=None, weights_in=None, weights=True, **call):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    B, S, H, _ = q.shape
    out = torch.full((B, S, H, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    lse = torch.full((B, H, S), float("nan"), device="cuda")
    w = torch.full((B, cache.HK, cache.capacity), -7.0, device="cuda") if weights else None
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    fmha_fwd_kv4(q, cache, out, causal=causal, counts=n, scale=scale, lse=lse, weights=w, weights_in=weights_in, **call)
    again = torch.full_like(out, float("nan"))
    fmha_fwd_kv4(q, cache, again, causal=causal, counts=n, scale=scale, weights=None if w is None else w.clone(), **call)
    torch.cuda.synchronize()
    ref, ref_lse, ref_w, spread, peak, size, doubt = (x.cpu() for x in R.attend(q.cpu(), cache.pool.cpu(), cache.table.cpu(), cache.lengths.cpu(), causal, counts, scale,
                                                                                None if weights_in is None else weights_in.cpu()))
    assert torch.equal(out, again)
    off = 128 * 2.0 ** -24 * size + 2.0 ** -21
    got = out.cpu().double()
    assert torch.isfinite(got).all()
    longest = max(1, int(cache.lengths.max()))
    room = 2.0 ** -9 * ref.abs() + spread * (2.0 ** -9 + 4 * off.permute(0, 2, 1)[..., None]) * 1.01 + (longest * 1.5 * 2.0 ** -25 * peak)[..., None] + 1e-38
    assert ((got - ref).abs() <= room).all(), ((got - ref).abs() / room).max()
    lse = lse.cpu().double()
    none = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, none)
    assert ((lse - ref_lse).abs()[~none] <= (off + 2.0 ** -22 * ref_lse.abs())[~none]).all()
    if weights:
        w = w.cpu().double()
        t = torch.arange(w.shape[-1])
        live = (t < cache.lengths.cpu()[:, None, None]).expand_as(w)
        assert (w[~live] == -7.0).all()
        room = 2 * (128 * 2.0 ** -24 * doubt + 2.0 ** -20 * ref_w.abs()) + 1e-30
        assert ((w - ref_w).abs() <= room)[live].all(), ((w - ref_w).abs() / room)[live].max()
    return out


SHAPES = [
    # lengths, HK, group, S, page
    ([1], 1, 1, 1, 16), ([2, 0, 1], 2, 4, 1, 16), ([15, 16, 17], 1, 8, 1, 16), ([31, 32, 33, 63, 64, 65], 2, 4, 1, 32), ([127, 128, 129], 2, 3, 1, 64), ([255, 257, 5], 1, 16, 1, 128),
    ([1000, 1, 0, 333], 2, 5, 1, 64), ([700], 1, 2, 1, 128), ([129, 48], 2, 12, 1, 16), ([300, 77], 2, 4, 2, 64), ([300, 3], 1, 4, 5, 32), ([511, 130], 2, 8, 3, 64), ([90], 1, 16, 2, 16),
    ([260, 33], 1, 4, 33, 64), ([140, 9], 1, 8, 40, 32), ([131], 2, 1, 131, 16), ([257, 64, 0], 1, 3, 64, 128), ([200], 1, 16, 17, 64), ([385, 129], 2, 7, 60, 64),
]


@pytest.mark.parametrize("lengths,HK,group,S,page", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_attention_and_weights(lengths, HK, group, S, page, causal):
    cache = make_cache(lengths, HK, page, seed=sum(lengths))
    check_attend(cache, queries(len(lengths), S, HK * group), causal)


def test_rows_that_stand_for_nothing():
    """counts between nothing and all rows, cut where they exceed the rows or the length, below 0 none."""
    cache = make_cache([100, 40, 3, 70, 0], 2, 32)
    check_attend(cache, queries(5, 6, 8), True, counts=[0, 4, 5, -3, 2])
    check_attend(cache, queries(5, 6, 8), False, counts=[6, 100, 1, 2, 0])
    check_attend(cache, queries(5, 50, 8), True, counts=[7, 40, 3, 50, 1])


def test_lengths_beyond_the_table_are_cut():
    cache = make_cache([64, 64], 1, 16)
    cache.lengths.copy_(torch.tensor([1000, -5], dtype=torch.int32))
    q = queries(2, 1, 4)
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    out = torch.full_like(q, float("nan"))
    fmha_fwd_kv4(q, cache, out)
    cache.lengths.copy_(torch.tensor([64, 0], dtype=torch.int32))
    same = torch.full_like(q, float("nan"))
    fmha_fwd_kv4(q, cache, same)
    assert torch.equal(out, same) and (out[1] == 0).all() and torch.isfinite(out).all()


@pytest.mark.parametrize("S", [1, 40])
def test_a_wider_table_changes_nothing_behind_the_length(S):
    lengths = [130, 50]
    a, b = make_cache(lengths, 2, 32, seed=3), make_cache(lengths, 2, 32, seed=3, width=200)
    b.table[:, 5:] = 0x7FFFFFFF
    q = queries(2, S, 8)
    out_a = check_attend(a, q)
    out_b = check_attend(b, q)
    assert torch.allclose(out_a.float(), out_b.float(), rtol=2.0 ** -7, atol=1e-3)


@pytest.mark.parametrize("S,group", [(1, 4), (3, 8), (48, 4)])
def test_scales_of_v_from_tiny_to_huge(S, group):
    """Tokens whose values differ by many binades, blocks of zeros among them, in any order."""
    def gain(g, n):
        per_token = torch.exp2(torch.randint(-30, 30, (n, 1), generator=g).float())
        per_block = torch.exp2(torch.randint(-6, 6, (n, 4), generator=g).float()) * (torch.rand(n, 4, generator=g) > 0.1)
        return per_token * per_block.repeat_interleave(32, 1)
    check_attend(make_cache([150, 70], 1, 16, seed=5, v_gain=gain), queries(2, S, group))


@pytest.mark.parametrize("v_exponent", [-126, -70, 60, 100, 120])
@pytest.mark.parametrize("S", [1, 36])
def test_values_at_the_ends_of_the_range(S, v_exponent):
    cache = make_cache([90], 1, 32, seed=6, v_gain=lambda g, n: torch.full((n, 1), 2.0 ** v_exponent))
    check_attend(cache, queries(1, S, 4))


@pytest.mark.parametrize("S", [1, 34])
def test_rows_that_grow_late(S):
    """Scores that rise along the sequence, so that the running reference moves again and again, and one key that takes all the weight."""
    def gain(g, n):
        return torch.linspace(0.1, 6, n)[:, None]
    q = queries(1, S, 4, gain=3.0)
    check_attend(make_cache([400], 1, 64, seed=7, k_gain=gain), q)
    cache = make_cache([400], 1, 64, seed=8)
    codes, scales, _ = R.encode((q[0, 0, 0].float() * 4).bfloat16().cpu()[None])
    c, s = R.record(cache.pool, int(cache.table[0, 3]), 0, 0)
    c[17], s[17] = codes[0].cuda(), scales[0].cuda()
    check_attend(cache, q)


@pytest.mark.parametrize("S", [1, 40])
def test_other_scales_and_zero_queries(S):
    cache = make_cache([200, 33], 2, 64, seed=9)
    q = queries(2, S, 8)
    check_attend(cache, q, scale=0.5)
    check_attend(cache, q, scale=1e-3)
    q[0] = 0
    q[1, :, 3] *= 2.0 ** -100
    check_attend(cache, q)
    check_attend(cache, queries(2, S, 8) * 2.0 ** 60, scale=2.0 ** -60 / math.sqrt(128))


@pytest.mark.parametrize("S", [1, 40])
def test_tokens_that_nobody_sees_may_hold_anything(S):
    """NaN scales in the K and V of a token that the causal mask hides: rows in front of it do not notice, the others are NaN."""
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    rows = max(S, 2)
    cache = make_cache([100], 1, 32, seed=10)
    q = queries(1, rows, 4)
    ref = R.attend(q.cpu(), cache.pool.cpu(), cache.table.cpu(), cache.lengths.cpu(), True)[0]
    for part in (0, 1):
        dirty = make_cache([100], 1, 32, seed=10)
        R.record(dirty.pool, int(dirty.table[0, 3]), 0, part)[1][3] = 255   # token 99, the last
        R.record(dirty.pool, int(dirty.table[0, 3]), 0, part)[0][3] = 0
        out = torch.empty_like(q)
        fmha_fwd_kv4(q, dirty, out)
        assert torch.isnan(out[0, -1]).all()
        assert torch.isfinite(out[0, :-1]).all()
        assert (out[0, :-1].cpu().double() - ref[0, :-1]).abs().max() < 0.02


@pytest.mark.parametrize("S", [1, 40])
def test_infinite_and_nan_queries_stay_in_their_rows(S):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    cache = make_cache([100], 1, 32, seed=11)
    q = queries(1, S, 4)
    good = torch.empty_like(q)
    fmha_fwd_kv4(q, cache, good)
    bad = q.clone()
    bad[0, 0, 1, 5] = float("nan")
    bad[0, 0, 2, 7] = float("inf")
    out = torch.empty_like(q)
    fmha_fwd_kv4(bad, cache, out)
    assert torch.isnan(out[0, 0, 1]).all() and torch.isnan(out[0, 0, 2]).any()
    keep = torch.ones(S, 4, dtype=torch.bool)
    keep[0, 1:3] = False
    assert torch.equal(out[0][keep.cuda()], good[0][keep.cuda()])


@pytest.mark.parametrize("S", [1, 40])
@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31])
def test_pages_outside_the_pool_are_never_followed(S, bad):
    from amdgpu_rustdsl_b200 import device_status, fmha_fwd_kv4
    cache = make_cache([100, 100], 1, 16, seed=12)
    q = queries(2, S, 4)
    good = torch.empty_like(q)
    fmha_fwd_kv4(q, cache, good)
    cache.table[0, 2] = bad
    out = torch.empty_like(q)
    fmha_fwd_kv4(q, cache, out)
    assert torch.isnan(out[0]).all()   # every row sees tokens 32 to 47
    assert torch.equal(out[1], good[1]) or torch.allclose(out[1].float(), good[1].float(), rtol=2.0 ** -7, atol=1e-3)
    assert device_status() == 0


@pytest.mark.parametrize("S", [1, 40])
def test_weights_accumulate(S):
    cache = make_cache([150, 60, 0], 2, 32, seed=13)
    q = queries(3, S, 8)
    g = torch.Generator().manual_seed(2)
    before = torch.rand(3, 2, cache.capacity, generator=g).cuda()
    before[0, :, 150:] = float("nan")   # behind the length
    n = min(S, 150)
    before[0, :, 150 - n:150] = float("nan")   # tokens that are new in a causal call
    check_attend(cache, q, True, weights_in=before)
    before = torch.rand(3, 2, cache.capacity, generator=g).cuda()
    check_attend(cache, q, False, weights_in=before)
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    out, apart, within = torch.empty_like(q), torch.full_like(before, -1), before.clone()
    fmha_fwd_kv4(q, cache, out, weights=apart, weights_in=before)
    fmha_fwd_kv4(q, cache, out, weights=within, weights_in=within)
    live = (torch.arange(cache.capacity).cuda() < cache.lengths[:, None, None]).expand_as(apart)
    assert torch.equal(apart[live], within[live]) and (apart[~live] == -1).all() and torch.equal(within[~live], before[~live])


@pytest.mark.parametrize("S", [1, 40])
def test_strided_queries_other_streams_and_graphs(S):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    cache = make_cache([200, 90], 2, 64, seed=14)
    wide = torch.zeros(2, S, 3, 8, 128, dtype=torch.bfloat16, device="cuda")
    q = queries(2, S, 8)
    wide[:, :, 1] = q
    good = check_attend(cache, q)
    assert torch.equal(check_attend(cache, wide[:, :, 1]), good)
    stacked = q.transpose(1, 2).contiguous().transpose(1, 2)   # [B, H, S, 128] in memory
    assert torch.equal(check_attend(cache, stacked), good)
    side = torch.cuda.Stream()
    late = torch.zeros_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)   # the queries arrive on the side stream only after a while
        late.copy_(q)
        out = torch.empty_like(q)
        fmha_fwd_kv4(late, cache, out)
    side.synchronize()
    assert torch.equal(out, good)
    out.zero_()
    fmha_fwd_kv4(q, cache, out, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, good)
    graph = torch.cuda.CUDAGraph()
    w = torch.zeros(2, 2, cache.capacity, device="cuda")
    with torch.cuda.stream(side):
        fmha_fwd_kv4(q, cache, out, weights=w)   # the stream's workspace exists before the capture
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        fmha_fwd_kv4(q, cache, out, weights=w)
    for n in (200, 137):
        cache.lengths[0] = n
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, check_attend(cache, q))


def test_a_pool_beyond_32_bits():
    """Pages more than 2^32 bytes apart."""
    from amdgpu_rustdsl_b200 import Kv4Cache, fmha_fwd_kv4, kv4_append, kv4_read
    page, HK = 128, 8
    pages = (5 << 30) // (HK * 136 * page)
    pool = torch.empty(pages, HK, 136 * page, dtype=torch.uint8, device="cuda")
    table = torch.tensor([[pages - 1, 0], [3, pages - 2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([200, 256], dtype=torch.int32, device="cuda")
    big = Kv4Cache(pool, table, lengths)
    small = Kv4Cache(torch.empty(4, HK, 136 * page, dtype=torch.uint8, device="cuda"), torch.tensor([[2, 0], [3, 1]], dtype=torch.int32, device="cuda"), lengths)
    g = torch.Generator(device="cuda").manual_seed(4)
    k, v = (torch.randn(2, 256, HK, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
    counts = torch.tensor([200, 256], dtype=torch.int32, device="cuda")
    got = []
    for cache in (big, small):
        kv4_append(cache, k, v, counts=counts)
        rk, rv = torch.empty_like(k), torch.empty_like(v)
        kv4_read(cache, rk, rv)
        out = []
        for S in (1, 40):
            q = queries(2, S, 32)
            out.append(torch.empty_like(q))
            fmha_fwd_kv4(q, cache, out[-1])
        got.append([rk, rv] + out)
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_many_tiles_against_a_plain_product():
    """Long sequences, cut between many CTAs, against the same sums in f64 on the GPU."""
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4, kv4_append, kv4_read
    for B, HK, H, L, S in ((1, 1, 4, 70001, 1), (3, 2, 16, 20011, 1), (1, 2, 8, 30003, 5), (1, 1, 8, 5000, 700), (2, 2, 2, 3001, 1500), (150, 8, 32, 100, 1)):
        from amdgpu_rustdsl_b200 import Kv4Cache, kv4_pool
        per = -(-L // 64)
        cache = Kv4Cache(kv4_pool(B * per, HK), torch.randperm(B * per, device="cuda").int().view(B, per), torch.full((B,), L, dtype=torch.int32, device="cuda"))
        g = torch.Generator(device="cuda").manual_seed(L)
        k, v = (torch.randn(B, L, HK, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
        kv4_append(cache, k, v)
        kv4_read(cache, k, v)
        q = (torch.randn(B, S, H, 128, generator=g, device="cuda") * 2).bfloat16()
        out, lse = torch.empty_like(q), torch.empty(B, H, S, device="cuda")
        w = torch.zeros(B, HK, cache.capacity, device="cuda")
        fmha_fwd_kv4(q, cache, out, lse=lse, weights=w)
        at = torch.arange(L - S, L, device="cuda")
        for b in {0, B - 1}:
            for hk in {0, HK - 1}:
                mass = torch.zeros(L, dtype=torch.float64, device="cuda")
                for h in range(hk * (H // HK), (hk + 1) * (H // HK)):
                    x = q[b, :, h].double() @ k[b, :, hk].double().T / math.sqrt(128)
                    x.masked_fill_(torch.arange(L, device="cuda") > at[:, None], -math.inf)
                    ref_lse = torch.logsumexp(x, 1)
                    p = torch.exp(x - ref_lse[:, None])
                    ref, spread = p @ v[b, :, hk].double(), p @ v[b, :, hk].double().abs()
                    mass += p.sum(0)
                    # sizes of 128 products of normal values: below 128 * 2 * 6 * 6 / sqrt(128) = 815
                    off = 128 * 2.0 ** -24 * 815
                    room = 2.0 ** -9 * ref.abs() + spread * (2.0 ** -9 + 4 * off) + L * 1.5 * 2.0 ** -25 * (p * v[b, :, hk].double().abs().amax(1)).amax(1, keepdim=True)
                    assert ((out[b, :, h].double() - ref).abs() <= room).all()
                    assert ((lse[b, h].double() - ref_lse).abs() <= off).all()
                assert ((w[b, hk, :L].double() - mass).abs() <= 2 * off * mass + 1e-30).all()


def test_back_to_back_calls_give_the_same():
    """Many launches without a wait between them, of work that is cut between CTAs in the middle of items: none stalls, all give the same bits."""
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    cache = make_cache([3000, 1500], 2, 64, seed=15)
    for S in (1, 4, 100, 300):
        q = queries(2, S, 8)
        first, out = torch.empty_like(q), torch.empty_like(q)
        fmha_fwd_kv4(q, cache, first)
        for _ in range(200):
            fmha_fwd_kv4(q, cache, out)
        torch.cuda.synchronize()
        assert torch.equal(out, first)


def test_append_rounds_every_bf16_value_as_the_definition_does():
    """All 65536 bf16 bit patterns, each as the largest of its block and beside a larger one; whole blocks of zeros; Inf and NaN."""
    from amdgpu_rustdsl_b200 import Kv4Cache, kv4_append, kv4_pool, kv4_read
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    g = torch.Generator().manual_seed(3)
    rows = [bits.view(-1, 128), bits[torch.randperm(65536, generator=g)].view(-1, 128)]
    finite = bits[torch.isfinite(bits.float())]
    near = finite[:, None].float() * torch.rand(len(finite), 31, generator=g)   # blocks whose largest is the value itself
    blocks = torch.cat([finite[:, None].float(), near], 1).bfloat16()
    rows.append(blocks[:len(blocks) // 4 * 4].reshape(-1, 128))
    rows.append((torch.randn(2048, 128, generator=g)).bfloat16())
    rows.append(torch.zeros(4, 128).bfloat16())
    x = torch.cat(rows)
    x = x[:len(x) // 2 * 2]
    n = len(x) // 2
    for page in (16, 64):
        width = -(-n // page)
        cache = Kv4Cache(kv4_pool(width, 1, page), torch.randperm(width).int()[None].cuda(), torch.tensor([n], dtype=torch.int32).cuda())
        k, v = x[:n].view(1, n, 1, 128).cuda(), x[n:].view(1, n, 1, 128).cuda()
        kv4_append(cache, k, v)
        got_k, got_v = torch.empty_like(k), torch.empty_like(v)
        kv4_read(cache, got_k, got_v)
        for part, (src, got) in enumerate(((x[:n], got_k), (x[n:], got_v))):
            codes, scales, value = R.encode(src)
            for i in range(width):
                c, s = R.record(cache.pool.cpu(), int(cache.table[0, i]), 0, part)
                m = min(page, n - i * page)
                assert torch.equal(s[:m], scales[i * page:i * page + m])
                assert torch.equal(c[:m], codes[i * page:i * page + m])
            got, value = got.cpu().view(n, 128), value.bfloat16()
            assert torch.equal(torch.isnan(got), torch.isnan(value)) and torch.equal(got.nan_to_num(0), value.nan_to_num(0))
            assert torch.equal(torch.signbit(got)[~torch.isnan(got)], torch.signbit(value)[~torch.isnan(value)])


@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_writes_its_tokens_and_nothing_else(page):
    """Ragged numbers of new tokens from strided rows, over page ends, onto bytes that must stay; a page outside the pool drops its tokens."""
    from amdgpu_rustdsl_b200 import Kv4Cache, kv4_append, kv4_read
    lengths, counts, S, HK = [130, 1, 0, 70, 33, 200], [9, 1, 3, 0, 40, -1], 9, 3
    new = [max(0, min(S, n, c)) for n, c in zip(lengths, counts)]
    cache = make_cache(lengths, HK, page, seed=21, garbage=0x5A)
    before = cache.pool.clone()
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(6, S, 4 + 2 * HK, 128, generator=g).bfloat16().cuda()
    k, v = qkv[:, :, 4:4 + HK], qkv[:, :, 4 + HK:]
    n_counts = torch.tensor(counts, dtype=torch.int32, device="cuda")
    lost = int(cache.table[0, 129 // page])
    cache.table[0, 129 // page] = 10 ** 6
    kv4_append(cache, k, v, counts=n_counts)
    expect, held = before.cpu().clone(), [torch.zeros(6, S, HK, 128, dtype=torch.bfloat16) for _ in range(2)]
    for b, m in enumerate(new):
        for i in range(m):
            t = lengths[b] - m + i
            gone = b == 0 and t // page == 129 // page
            for h in range(HK):
                for part, x in ((0, k), (1, v)):
                    codes, scales, value = R.encode(x[b, i, h].cpu()[None])
                    if gone:
                        held[part][b, i, h] = float("nan")
                        continue
                    c, s = R.record(expect, int(cache.table[b, t // page]), h, part)
                    c[t % page], s[t % page] = codes[0], scales[0]
                    held[part][b, i, h] = value[0].bfloat16()
    assert torch.equal(cache.pool.cpu(), expect)
    got = [torch.full((6, S, HK, 128), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    kv4_read(cache, got[0], got[1], last=True, counts=n_counts)
    for a, e in zip(got, held):
        a = a.cpu()
        assert torch.equal(torch.isnan(a), torch.isnan(e)) and torch.equal(a.nan_to_num(0), e.nan_to_num(0))
    cache.table[0, 129 // page] = lost
    kv4_append(cache, k, v)   # without counts: as many as there are, up to the length
    kv4_read(cache, got[0], got[1], last=True)
    for part, x in ((0, k), (1, v)):
        for b, n in enumerate(lengths):
            m = min(S, n)
            value = R.encode(x[b, :m].cpu().reshape(-1, 128))[2].view(m, HK, 128).bfloat16()
            assert torch.equal(got[part][b, :m].cpu(), value) and (got[part][b, m:] == 0).all()


def test_read_from_the_start_and_into_strided_rows():
    from amdgpu_rustdsl_b200 import kv4_read
    lengths = [70, 0, 5]
    cache = make_cache(lengths, 2, 32, seed=22)
    wide = torch.full((3, 80, 5, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    kv4_read(cache, wide[:, :, 0:2], wide[:, :, 3:5])
    assert (wide[:, :, 2] == 9).all()
    for b, n in enumerate(lengths):
        for h in range(2):
            k, v = R.tokens(cache.pool.cpu(), cache.table[b].tolist(), h, n)
            assert torch.equal(wide[b, :n, h].cpu().double(), k) and torch.equal(wide[b, :n, 3 + h].cpu().double(), v)
        assert (wide[b, n:, :2] == 0).all() and (wide[b, n:, 3:] == 0).all()


def check_evict(cache, weights, keep, recent, first, seed=0, same_pool=False):
    from amdgpu_rustdsl_b200 import Kv4Cache, kv4_evict
    B, HK, page = cache.B, cache.HK, cache.page
    per = -(-keep // page)
    pool = torch.full((B * per + 2, HK, 136 * page), 0x33, dtype=torch.uint8, device="cuda")
    table = torch.randperm(B * per + 2)[:B * per].int().view(B, per).cuda()
    if same_pool:
        table += cache.pool.shape[0]
        cache = Kv4Cache(torch.cat([cache.pool, pool]), cache.table, cache.lengths)
        pool = cache.pool
    into = Kv4Cache(pool, table, torch.full((B,), -1, dtype=torch.int32, device="cuda"))
    before = pool.cpu().clone()
    kept = torch.full((B, HK, keep), -9, dtype=torch.int32, device="cuda")
    out = torch.full((B, HK, keep + 3), -9.0, device="cuda")
    kv4_evict(cache, weights, into, keep=keep, recent=recent, first=first, kept=kept, weights_out=out)
    stay = R.evict(weights.cpu(), cache.lengths.cpu(), keep, recent, first)
    assert into.lengths.tolist() == [min(int(n), keep) for n in cache.lengths.cpu()]
    source, expect, w, out = cache.pool.cpu() if not same_pool else before, before, weights.cpu(), out.cpu()
    for b in range(B):
        for h in range(HK):
            s = stay[b][h]
            assert kept[b, h].tolist() == s + [-1] * (keep - len(s))
            at = torch.tensor(s, dtype=torch.long)
            a, e = out[b, h, :len(s)], w[b, h][at]
            assert torch.equal(a.view(torch.int32), e.view(torch.int32)) and (out[b, h, len(s):] == -9).all()
            for j, t in enumerate(s):
                for part in (0, 1):
                    c, sc = R.record(source, int(cache.table[b, t // page]), h, part)
                    ec, es = R.record(expect, int(table[b, j // page]), h, part)
                    ec[j % page], es[j % page] = c[t % page], sc[t % page]
    assert torch.equal(into.pool.cpu(), expect)
    # without the optional outputs the cache is the same
    again = Kv4Cache(torch.full_like(pool, 0x33), table, torch.zeros(B, dtype=torch.int32, device="cuda"))
    kv4_evict(cache, weights, again, keep=keep, recent=recent, first=first)
    if not same_pool:
        assert torch.equal(again.pool, into.pool) and torch.equal(again.lengths, into.lengths)


@pytest.mark.parametrize("lengths,HK,page,keep,recent,first", [
    ([1], 1, 16, 1, 0, 0), ([0, 1, 2], 2, 16, 1, 0, 0), ([5, 40, 17], 2, 16, 16, 4, 2), ([100, 33, 0], 3, 32, 33, 33, 0), ([100, 90], 1, 64, 20, 0, 20), ([300, 299, 301], 2, 128, 300, 10, 4),
    ([1025, 2049, 1023], 1, 64, 500, 64, 4), ([3000], 2, 128, 2999, 0, 0), ([700, 65], 2, 16, 64, 1, 1)])
def test_eviction(lengths, HK, page, keep, recent, first):
    cache = make_cache(lengths, HK, page, seed=31)
    g = torch.Generator().manual_seed(6)
    w = torch.exp2(torch.randn(len(lengths), HK, cache.capacity + 5, generator=g) * 4)
    check_evict(cache, w.cuda(), keep, recent, first)


def test_eviction_of_equal_negative_infinite_and_nan_weights():
    lengths, HK = [400, 400, 400, 400, 400], 1
    cache = make_cache(lengths, HK, 64, seed=32)
    g = torch.Generator().manual_seed(7)
    w = torch.randn(5, 1, cache.capacity, generator=g)
    w[0] = 0.25                                                     # all equal: the earliest
    w[1] = torch.randint(0, 3, w[1].shape, generator=g).float()     # few values
    w[1][w[1] == 0] *= torch.sign(torch.randn(int((w[1] == 0).sum()), generator=g))   # zeros of both signs are equal
    w[2, 0, ::3], w[2, 0, 1::7], w[2, 0, 5::11] = math.inf, -math.inf, math.nan
    w[3, 0, ::2] = torch.tensor([-1], dtype=torch.int32).view(torch.float32)   # NaN with the sign bit
    w[4] = torch.randint(0, 40, w[4].shape, generator=g).float() * 2.0 ** -149   # subnormal
    for keep, recent, first in ((100, 0, 0), (100, 30, 5), (399, 0, 0)):
        check_evict(cache, w.cuda(), keep, recent, first)


def test_eviction_within_one_pool_and_of_pages_outside_it():
    from amdgpu_rustdsl_b200 import Kv4Cache, kv4_evict, kv4_read
    cache = make_cache([200, 90], 2, 32, seed=33)
    w = torch.rand(2, 2, cache.capacity, generator=torch.Generator().manual_seed(8)).cuda()
    check_evict(cache, w, 50, 10, 2, same_pool=True)
    cache.table[0, 1] = 1 << 20   # tokens 32 to 63 are lost: they read as NaN where they stay
    w[0, :, 32:64] = 5.0
    into = Kv4Cache(torch.zeros(4, 2, 136 * 32, dtype=torch.uint8, device="cuda"), torch.tensor([[0, 1], [2, -7]], dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"))
    kv4_evict(cache, w, into, keep=40)
    k, v = (torch.empty(2, 40, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kv4_read(into, k, v)
    nan = torch.isnan(k[0, :, 0]).all(-1)
    assert int(nan.sum()) == 32 and torch.equal(torch.isnan(v[0, :, 0]).all(-1), nan) and torch.isfinite(k[1, :32].float()).all() and torch.isnan(k[1, 32:]).all()


def test_refusals_of_the_python_entry():
    from amdgpu_rustdsl_b200 import Kv4Cache, fmha_fwd_kv4, kv4_append, kv4_evict, kv4_read
    cache = make_cache([40, 20], 2, 16, seed=41)
    q = queries(2, 1, 8)
    out = torch.empty_like(q)
    for bad, message in ((q.float(), "bf16"), (q[..., :64], "bf16"), (q[:1], "bf16"), (q.cpu(), "device"), (q.transpose(2, 3).contiguous().transpose(2, 3), "dense")):
        with pytest.raises(ValueError, match=message):
            fmha_fwd_kv4(bad, cache, out)
    odd = torch.empty(2 * 8 * 128 + 8, dtype=torch.bfloat16, device="cuda")[4:-4].view(2, 1, 8, 128)
    with pytest.raises(ValueError, match="16 bytes"):
        fmha_fwd_kv4(odd, cache, out)
    for bad in (out.float(), out[:, :, :4], torch.empty(2, 8, 1, 128, dtype=torch.bfloat16, device="cuda").transpose(1, 2).expand(2, 1, 8, 128)[:, :, ::1].transpose(0, 1)):
        with pytest.raises(ValueError):
            fmha_fwd_kv4(q, cache, bad)
    with pytest.raises(ValueError, match="1 to 16 times"):
        fmha_fwd_kv4(queries(2, 1, 34), cache, torch.empty(2, 1, 34, 128, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError, match="1 to 16 times"):
        fmha_fwd_kv4(queries(2, 1, 3), cache, torch.empty(2, 1, 3, 128, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError, match="counts"):
        fmha_fwd_kv4(q, cache, out, counts=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="lse"):
        fmha_fwd_kv4(q, cache, out, lse=torch.empty(2, 1, 8, device="cuda"))
    with pytest.raises(ValueError, match="weights"):
        fmha_fwd_kv4(q, cache, out, weights=torch.empty(2, 2, cache.capacity - 1, device="cuda"))
    with pytest.raises(ValueError, match="without weights"):
        fmha_fwd_kv4(q, cache, out, weights_in=torch.empty(2, 2, cache.capacity, device="cuda"))
    with pytest.raises(ValueError, match="scale"):
        fmha_fwd_kv4(q, cache, out, scale=-1.0)
    k = torch.empty(2, 3, 2, 128, dtype=torch.bfloat16, device="cuda")
    for args in ((k, k[:, :2]), (k[:, :, :1], k), (k.half(), k)):
        with pytest.raises(ValueError):
            kv4_append(cache, *args)
        with pytest.raises(ValueError):
            kv4_read(cache, *args)
    with pytest.raises(ValueError, match="counts"):
        kv4_read(cache, k, k, counts=cache.lengths)
    w = torch.zeros(2, 2, cache.capacity, device="cuda")
    into = Kv4Cache(cache.pool, cache.table.clone(), torch.zeros_like(cache.lengths))
    for call in (dict(keep=0), dict(keep=cache.capacity + 1), dict(keep=4, recent=3, first=2), dict(keep=4, recent=-1), dict(keep=4, kept=torch.zeros(2, 2, 5, dtype=torch.int32, device="cuda")),
                 dict(keep=4, weights_out=torch.zeros(2, 2, 3, device="cuda"))):
        with pytest.raises(ValueError):
            kv4_evict(cache, w, into, **call)
    with pytest.raises(ValueError, match="of its own"):
        kv4_evict(cache, w, cache, keep=4)
    with pytest.raises(ValueError):
        kv4_evict(cache, w[:, :, :-1], into, keep=4)
