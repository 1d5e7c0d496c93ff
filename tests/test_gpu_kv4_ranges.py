"""Keys and queries far from 1 over the 4-bit cache, within the ranges that the C header names (tolerances as in test_gpu_kv4.py)."""
import math

import pytest
import torch

from tests.test_gpu_kv4 import check_attend, make_cache, no_wait_ran_out, queries  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k_exponent,q_exponent", [(90, 0), (90, -90), (-100, 0), (-100, 60), (-60, 100), (0, 100), (0, -90), (20, 100), (98, 20)])
@pytest.mark.parametrize("S", [1, 3, 6, 40])
def test_keys_and_queries_of_any_size(S, k_exponent, q_exponent):
    """The scale brings the scores back to the ordinary."""
    cache = make_cache([150, 33], 1, 16, seed=95, k_gain=lambda g, n: torch.full((n, 1), 2.0 ** k_exponent))
    check_attend(cache, queries(2, S, 4) * 2.0 ** q_exponent, scale=2.0 ** -(k_exponent + q_exponent) / math.sqrt(128))


@pytest.mark.parametrize("S", [1, 6, 40])
def test_keys_of_many_sizes_in_one_sequence(S):
    """Tokens of 2^-12 to 2^2: the small ones weigh alike."""
    def gain(g, n):
        return torch.exp2(torch.randint(-12, 2, (n, 1), generator=g).float())
    check_attend(make_cache([400, 129], 2, 64, seed=96, k_gain=gain), queries(2, S, 8))
