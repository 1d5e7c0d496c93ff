"""The 4-bit cache where a CTA has much to do: rings that are refilled many times. Against 64 bits on the GPU.

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


# rows of a KV head from one group of eight to four, pages of every size; lengths off the tiles of 128, and enough of them for a dozen tiles a CTA
@pytest.mark.parametrize("S,group,page,causal", [(1, 4, 16, True), (1, 8, 128, True), (2, 4, 32, False), (3, 4, 16, True), (4, 4, 128, True), (5, 4, 64, True), (3, 8, 16, False), (8, 4, 16, True),
                                                 (2, 16, 128, True), (12, 4, 32, True)])
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
