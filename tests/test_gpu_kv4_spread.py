"""Attention over the 4-bit cache where V's scales differ by up to the 224 binades that the kernels tell apart: a softmax sum knows nothing of them.

Tolerances are those of test_gpu_kv4.py, with what large exponents add: as in test_gpu_kv8_spread.py eight roundings of numbers below 2^9, 2^-16 each, `WIDE`, to a log-sum-exp and, doubled, to a weight."""
import math

import pytest
import torch

from tests import kv4_reference as R
from tests import test_gpu_kv4 as K
from tests.test_gpu_kv4 import no_wait_ran_out  # noqa: F401
from tests.test_gpu_kv8_spread import PATTERNS, WIDE

pytestmark = pytest.mark.gpu


def gains(pattern, turns, rows):
    """V's sizes by units: the pattern over the sequence's length, or `turns` times. (Units are tokens whose factors are taken relative to their largest: within them V is exact down to 2^-33 of that only.)"""
    unit = 32 if rows <= 32 else 128

    def gain(g, n):
        units = -(-n // unit)
        at = [pattern[u * len(pattern) * turns // max(units, len(pattern)) % len(pattern)] for u in range(units)]
        return torch.tensor([0.0 if e is None else 2.0 ** e for e in at]).repeat_interleave(unit)[:n, None]
    return gain


def check(cache, q, causal):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    B, S, H, _ = q.shape
    out, lse = torch.full_like(q, float("nan")), torch.full((B, H, S), float("nan"), device="cuda")
    w = torch.zeros(B, cache.HK, cache.capacity, device="cuda")
    fmha_fwd_kv4(q, cache, out, causal=causal, lse=lse, weights=w)
    ref, ref_lse, ref_w, spread, peak, size, doubt = (x.cpu() for x in R.attend(q.cpu(), cache.pool.cpu(), cache.table.cpu(), cache.lengths.cpu(), causal, None, None, None))
    off = 128 * 2.0 ** -24 * size + 2.0 ** -21 + WIDE
    none, lse = ref_lse == -math.inf, lse.cpu().double()
    assert torch.equal(lse == -math.inf, none)
    assert ((lse - ref_lse).abs()[~none] <= (off + 2.0 ** -22 * ref_lse.abs())[~none]).all(), (lse - ref_lse).abs()[~none].max()
    longest = max(1, int(cache.lengths.max()))
    room = 2.0 ** -9 * ref.abs() + spread * (2.0 ** -9 + 4 * off.permute(0, 2, 1)[..., None]) * 1.01 + (longest * 1.5 * 2.0 ** -25 * peak)[..., None] + 1e-38
    assert ((out.cpu().double() - ref).abs() <= room).all()
    live = (torch.arange(w.shape[-1]) < cache.lengths.cpu()[:, None, None]).expand_as(w.cpu())
    assert ((w.cpu().double() - ref_w).abs() <= 2 * (128 * 2.0 ** -24 * doubt + (2.0 ** -20 + WIDE) * ref_w.abs()) + 1e-30)[live].all()


SHAPES = [
    # lengths, HK, group, S, page: one CTA's, many CTAs' with a step each, more steps than CTAs
    ([100], 1, 4, 1, 16), ([128, 33], 2, 8, 3, 32), ([130], 1, 16, 2, 128), ([3000], 1, 4, 1, 64), ([1500, 900], 1, 16, 2, 16), ([3000] * 8, 4, 4, 1, 64), ([2000] * 8, 4, 5, 2, 64), ([2000] * 6, 4, 6, 3, 32),
    ([1500] * 6, 4, 16, 2, 32), ([150, 47], 1, 4, 36, 16), ([3000], 1, 4, 40, 64), ([1100, 700], 1, 8, 100, 32), ([700, 650, 701, 600], 8, 1, 40, 64), ([500] * 20, 4, 1, 40, 128),
]


@pytest.mark.parametrize("lengths,HK,group,S,page", SHAPES)
@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("turns", [1, 3])
def test_sums_know_nothing_of_the_values(lengths, HK, group, S, page, pattern, turns):
    check(K.make_cache(lengths, HK, page, seed=len(pattern), v_gain=gains(pattern, turns, S * group)), K.queries(len(lengths), S, HK * group), S % 2 == 0)


@pytest.mark.parametrize("S", [1, 40])
def test_values_of_zero_leave_the_sum_to_the_others(S):
    """Half of the tokens have the scores of the other half and values of zero: outputs are half of the others' mean."""
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4, kv4_read
    B, n = 200, 256
    cache = K.make_cache([n] * B, 2, 64, seed=1, k_gain=lambda g, n: torch.zeros(n, 1), v_gain=lambda g, n: torch.cat([torch.zeros(n // 2, 1), torch.full((n // 2, 1), 2.0 ** 100)]))
    q = K.queries(B, S, 2)
    out, lse, k, v = torch.empty_like(q), torch.empty(B, 2, S, device="cuda"), *(torch.empty(B, n, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    fmha_fwd_kv4(q, cache, out, causal=False, lse=lse)
    kv4_read(cache, k, v)
    v = v.double()
    assert ((lse.double() - math.log(n)).abs() <= WIDE).all()
    assert ((out.double() - v.mean(1)[:, None]).abs() <= (2.0 ** -8 + 2.0 ** -9 + WIDE) * v.abs().mean(1)[:, None]).all()
