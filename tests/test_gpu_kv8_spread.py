"""Attention over the 8-bit cache where V's scales differ by up to the 209 binades that they may: a softmax sum knows nothing of them.

Tolerances are those of test_gpu_kv8.py, with what large exponents add. The kernels' exponents, references and their differences stay below 2^9 in size here, where a rounding is 2^-16 at most; a weight or
a sum goes through eight of them at most (argument, its fma, half and whole of two changes of reference, the merges of warps and of CTAs, the logarithm), in base 2: `wide` is 2^-13."""
import math

import pytest
import torch

from tests import kv8_reference as R
from tests import test_gpu_kv8 as K
from tests.test_gpu_kv8 import no_wait_ran_out  # noqa: F401

pytestmark = pytest.mark.gpu

WIDE = 2.0 ** -13

# exponents of V's size, None for values of zero (whose scale is 2^-90)
PATTERNS = [(None, 60), (60, None), (-70, 120), (120, -70), (120, None, 0, None), (None, -70, 0, 60, 120)]


def gains(pattern, turns):
    """V's sizes by block: the pattern over the sequence's length, or `turns` times."""
    def gain(g, n):
        blocks = -(-n // 16)
        at = [pattern[b * len(pattern) * turns // blocks % len(pattern)] for b in range(blocks)]
        return torch.tensor([0.0 if e is None else 2.0 ** e for e in at]).repeat_interleave(16)[:n]
    return lambda g, n: gain(g, n)[:, None]


def check(cache, q, causal):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv8
    out, lse = torch.full_like(q, float("nan")), torch.full((q.shape[0], q.shape[2], q.shape[1]), float("nan"), device="cuda")
    fmha_fwd_kv8(q, cache, out, causal=causal, lse=lse)
    ref, ref_lse, spread, peak, size = R.attend(q.cpu(), cache.pool.cpu(), cache.table.cpu(), cache.lengths.tolist(), causal)
    none = ref_lse == -math.inf
    room, lse_room = K.room_of(ref, spread, peak, size, ref_lse.masked_fill(none, 0.0), max(1, int(cache.lengths.max())))
    lse = lse.cpu().double()
    assert torch.equal(lse == -math.inf, none)
    assert ((lse - ref_lse).abs()[~none] <= lse_room[~none] + WIDE).all(), (lse - ref_lse).abs()[~none].max()
    assert ((out.cpu().double() - ref).abs() <= room + 4 * WIDE * spread).all()


SHAPES = [
    # lengths, HK, group, S, page: whole items and items of many parts, of each kernel
    ([90], 1, 4, 1, 16), ([200, 33], 2, 8, 3, 32), ([130], 1, 16, 2, 128), ([3000], 1, 4, 1, 64), ([1500, 900], 1, 16, 2, 16), ([9000], 1, 2, 1, 64), ([150, 47], 1, 4, 36, 16), ([3000], 1, 4, 40, 64),
    ([2100, 700], 1, 8, 100, 32),
]


@pytest.mark.parametrize("lengths,HK,group,S,page", SHAPES)
@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("turns", [1, 3])
def test_sums_know_nothing_of_the_values(lengths, HK, group, S, page, pattern, turns):
    cache = K.make_cache(lengths, HK, page, seed=len(pattern), v_gain=gains(pattern, turns))
    check(cache, K.queries(len(lengths), S, HK * group), S % 2 == 0)


@pytest.mark.parametrize("pattern", PATTERNS[:4])
def test_prompts_whose_parts_lie_by_columns(pattern):
    """32 items among the CTAs, each cut in a few parts."""
    cache = K.make_cache([700, 650, 701, 600], 8, 64, seed=5, v_gain=gains(pattern, 1))
    check(cache, K.queries(4, 40, 8), True)


@pytest.mark.parametrize("S", [1, 40])
def test_values_of_zero_leave_the_sum_to_the_others(S):
    """Half of the tokens have the scores of the other half and values of zero: outputs are half of the others' mean."""
    from amdgpu_rustdsl_b200 import fmha_fwd_kv8
    cache = K.make_cache([64], 1, 64, seed=1, k_gain=lambda g, n: torch.zeros(n, 1), v_gain=lambda g, n: torch.cat([torch.zeros(32, 1), torch.full((32, 1), 2.0 ** 100)]))
    q = K.queries(1, S, 4)
    out, lse = torch.empty_like(q), torch.empty(1, 4, S, device="cuda")
    fmha_fwd_kv8(q, cache, out, causal=False, lse=lse)
    _, v, _ = R.tokens(cache.pool.cpu(), cache.table.cpu(), 0, 0, 64)
    assert ((lse.cpu().double() - math.log(64)).abs() <= WIDE).all()
    assert ((out.cpu().double() - v.mean(0)).abs() <= (2.0 ** -8 + 2.0 ** -11 + WIDE) * v.abs().mean(0)).all()
