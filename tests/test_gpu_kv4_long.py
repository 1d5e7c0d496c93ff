"""The 4-bit cache where a CTA has much to do: rings that are refilled many times, selections of many rounds. Against 64 bits on the GPU.

Tolerances. A score is off by at most 128 * 2^-24 of the sum of its products' sizes, exp2 and log2 by 2^-21 (`off`). A sum over L tokens in f32 is off by L * 2^-24 of
the sum of its terms' sizes at most. An output has two such scores and sums, weights rounded to f16 (2^-11; below 2^-24 of the row's largest product they vanish,
1.5 * 2^-25 of it per token) and is rounded to bf16 (2^-8)."""
import math

import pytest
import torch

from tests.test_gpu_kv4 import no_wait_ran_out  # noqa: F401

pytestmark = pytest.mark.gpu


def filled(lengths, HK, page, seed, width=None):
    """A cache filled by append, and the values it holds, f64 [B, longest, HK, 128]."""
    from amdgpu_rustdsl_b200 import Kv4Cache, kv4_append, kv4_pool, kv4_read
    B, longest = len(lengths), max(lengths)
    width = -(-longest // page) if width is None else width
    used = -(-longest // page)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    table[:, :used] = torch.randperm(B * used, device="cuda").int().view(B, used)
    cache = Kv4Cache(kv4_pool(B * used, HK, page), table, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    g = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.randn(B, longest, HK, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
    kv4_append(cache, k, v, counts=cache.lengths)
    kv4_read(cache, k, v)
    return cache, k, v


# rows of a KV head from one group of eight to four, and for the tensor cores' tiles; pages of every size; lengths off the tiles of 128, and enough of them for a dozen tiles a CTA
@pytest.mark.parametrize("S,group,page,causal", [(1, 4, 16, True), (1, 8, 128, True), (2, 4, 32, False), (3, 4, 16, True), (4, 4, 128, True), (5, 4, 64, True), (3, 8, 16, False), (8, 4, 16, True),
                                                 (2, 16, 128, True), (12, 4, 32, True), (70, 4, 64, True), (9, 5, 16, False)])
def test_many_tiles_a_cta(S, group, page, causal):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    lengths, HK = [8001, 7937, 8063, 8000, 7000, 8064, 5555, 8050, 8033, 8011, 7999, 8003, 6003, 8039, 8040, 7777], 8
    cache, k, v = filled(lengths, HK, page, S * group)
    B, H = len(lengths), HK * group
    g = torch.Generator(device="cuda").manual_seed(9)
    q = (torch.randn(B, S, H, 128, generator=g, device="cuda") * torch.exp2(torch.rand(H, 1, generator=g, device="cuda") * 2 - 1)).bfloat16()
    out, lse = torch.full_like(q, math.nan), torch.full((B, H, S), math.nan, device="cuda")
    weights, weights_in = torch.full((B, HK, cache.capacity), -7.0, device="cuda"), torch.rand(B, HK, cache.capacity, generator=g, device="cuda")
    fmha_fwd_kv4(q, cache, out, causal=causal, lse=lse, weights=weights, weights_in=weights_in)
    for b, L in enumerate(lengths):
        sees = torch.arange(L, device="cuda") <= (torch.arange(L - S, L, device="cuda") if causal else torch.full((S,), L, device="cuda"))[:, None]
        sees = sees.repeat_interleave(group, 0)
        for hk in range(HK):
            rows = q[b, :, hk * group:(hk + 1) * group].reshape(S * group, 128).double()
            keys, values = k[b, :L, hk].double(), v[b, :L, hk].double()
            x = (rows @ keys.T / math.sqrt(128)).masked_fill(~sees, -math.inf)
            off = 128 * 2.0 ** -24 * (rows.abs() @ keys.abs().T / math.sqrt(128)).amax(1) + 2.0 ** -21
            ref_lse = torch.logsumexp(x, 1)
            p = torch.exp(x - ref_lse[:, None])
            ref, spread, peak = p @ values, p @ values.abs(), (p * values.abs().amax(1)).amax(1)
            got = out[b, :, hk * group:(hk + 1) * group].reshape(S * group, 128).double()
            room = 2.0 ** -8 * ref.abs() + spread * (2.0 ** -11 + 4 * off[:, None] + 2 * L * 2.0 ** -24) * 1.01 + (L * 1.5 * 2.0 ** -25 * peak)[:, None]
            assert ((got - ref).abs() <= room).all(), (b, hk, ((got - ref).abs() / room).max())
            got = lse[b, hk * group:(hk + 1) * group].T.reshape(-1).double()
            assert ((got - ref_lse).abs() <= off + L * 2.0 ** -24 + 2.0 ** -22 * ref_lse.abs()).all(), (b, hk)
            old = weights_in[b, hk, :L].double()
            if causal:
                old[L - S:] = 0
            mass = p.sum(0)
            room = 2 * (p * (off + L * 2.0 ** -24)[:, None]).sum(0) + 2.0 ** -20 * (mass + old) + 1e-30
            got = weights[b, hk].double()
            assert ((got[:L] - mass - old).abs() <= room).all() and (got[L:] == -7.0).all(), (b, hk)


def check_evict(lengths, HK, page, keep, recent, first, weights, width=None):
    """Positions by a stable sort, weights and values gathered from them."""
    from amdgpu_rustdsl_b200 import Kv4Cache, kv4_evict, kv4_pool, kv4_read
    B, per = len(lengths), -(-keep // page)
    cache, k, v = filled(lengths, HK, page, keep, width)
    weights = weights(B, HK, cache.capacity)
    into = Kv4Cache(kv4_pool(B * per, HK, page), torch.randperm(B * per, device="cuda").int().view(B, per), torch.full((B,), -1, dtype=torch.int32, device="cuda"))
    kept, out = torch.full((B, HK, keep), -9, dtype=torch.int32, device="cuda"), torch.full((B, HK, keep), -9.0, device="cuda")
    kv4_evict(cache, weights, into, keep=keep, recent=recent, first=first, kept=kept, weights_out=out)
    new_k, new_v = (torch.empty(B, keep, HK, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kv4_read(into, new_k, new_v)
    assert into.lengths.tolist() == [min(n, keep) for n in lengths]
    for b, L in enumerate(lengths):
        for h in range(HK):
            stay = torch.arange(min(L, keep), device="cuda")
            if L > keep:
                some = weights[b, h, first:L - recent] + 0.0   # (zeros of either sign are equal)
                order = torch.sort(some.cpu(), descending=True, stable=True).indices[:keep - first - recent].cuda() + first
                stay = torch.cat([torch.arange(first, device="cuda"), order.sort().values, torch.arange(L - recent, L, device="cuda")])
            n = len(stay)
            assert torch.equal(kept[b, h, :n].long(), stay) and (kept[b, h, n:] == -1).all(), (b, h)
            assert torch.equal(out[b, h, :n].view(torch.int32), weights[b, h, stay].view(torch.int32)) and (out[b, h, n:] == -9).all()
            assert torch.equal(new_k[b, :n, h], k[b, stay, h]) and torch.equal(new_v[b, :n, h], v[b, stay, h]), (b, h)


def few_values(B, HK, n):
    """Many equal weights, so that the cut lies among equals that every round and CTA has some of."""
    return torch.randint(0, 6, (B, HK, n), generator=torch.Generator(device="cuda").manual_seed(n), device="cuda").float()


def long_tailed(B, HK, n):
    g = torch.Generator(device="cuda").manual_seed(n + 1)
    w = torch.exp2(torch.randn(B, HK, n, generator=g, device="cuda") * 3) * (torch.rand(B, HK, n, generator=g, device="cuda") > 0.1)
    w[:, :, ::977], w[:, :, 5::1993], w[:, :, 7::1501] = math.nan, -math.inf, math.inf
    return w


@pytest.mark.parametrize("weights", [few_values, long_tailed])
@pytest.mark.parametrize("lengths,HK,page,keep,recent,first,width", [
    # one CTA a head, 8 to 16 rounds of 512 tokens
    ([4096, 8000, 8191, 4097, 5003, 7168, 512, 513, 1, 0, 6000, 8192, 7777, 4608, 4607, 3000], 8, 64, 1024, 128, 4, None),
    ([8192, 6001, 5000], 64, 32, 4900, 0, 0, None),
    # 8 CTAs a head, 13 rounds each, and sequences of which some CTAs have a round or none
    ([50001, 4000, 37], 8, 128, 6250, 500, 16, None),
    ([65536, 65535], 2, 128, 30000, 1, 1, None),
    # tables of more than 65536 tokens: keys that are read again, with one round a CTA and with up to 37
    ([3000, 66000, 5], 2, 128, 1000, 10, 3, 520),
    ([150000, 70001], 2, 64, 40000, 0, 0, None),
])
def test_evictions_of_many_rounds(lengths, HK, page, keep, recent, first, width, weights):
    check_evict(lengths, HK, page, keep, recent, first, weights, width)


@pytest.mark.parametrize("S,weights", [(1, True), (2, True), (3, False), (8, False), (70, False)])
def test_attention_in_place(S, weights):
    """out may be q, cut items and sequences without tokens among them."""
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    cache, _, _ = filled([5000, 1, 3001, 777], 2, 32, S)
    cache.lengths[1] = 0
    g = torch.Generator(device="cuda").manual_seed(S)
    q = torch.randn(4, S, 8, 128, generator=g, device="cuda").bfloat16()
    out, w, v = torch.full_like(q, math.nan), *(torch.zeros(4, 2, cache.capacity, device="cuda") for _ in range(2))
    fmha_fwd_kv4(q, cache, out, weights=w if weights else None)
    fmha_fwd_kv4(q, cache, q, weights=v if weights else None)
    assert torch.equal(q, out) and torch.equal(w, v)
