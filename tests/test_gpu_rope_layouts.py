"""Rotary positions: queries and keys that lie between one another without sharing an element, and every form of rows at numbers of tokens that share a CTA (reference and tolerances: test_gpu_rope.py)."""
import math

import pytest
import torch

from tests import test_gpu_rope as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,S", [(1, 1), (2, 1), (1, 7), (2, 7), (3, 333)])
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("where", ["heads first", "tokens first", "tokens outermost"])
def test_queries_and_keys_of_one_projection(B, S, backward, where):
    from amdgpu_rustdsl_b200 import Rope, rope_rotate
    H, HK, D = 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(B + S)
    order = {"heads first": (0, 2, 1, 3), "tokens first": (0, 1, 2, 3), "tokens outermost": (1, 0, 2, 3)}[where]
    rows = torch.randn(B, S, H + 2 * HK, D, generator=g, device="cuda").bfloat16()
    qkv = torch.empty([rows.shape[i] for i in order], dtype=torch.bfloat16, device="cuda").permute([order.index(i) for i in range(4)])
    qkv.copy_(rows)
    rope, at = Rope(64), torch.randint(0, 9000, (B, S), generator=g, device="cuda")
    q, k = (torch.empty(B, S, n, D, dtype=torch.bfloat16, device="cuda") for n in (H, HK))
    rope_rotate(rope, rows[:, :, :H], at, q, backward=backward)
    rope_rotate(rope, rows[:, :, H:H + HK], at, k, backward=backward)
    rope_rotate(rope, qkv[:, :, :H], at, y=qkv[:, :, H:H + HK], backward=backward)
    assert torch.equal(qkv, torch.cat([q, k, rows[:, :, H + HK:]], 2))


@pytest.mark.parametrize("type", R.TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("head,rotary,H,HK", [(128, 128, 5, 2), (128, 64, 32, 8), (96, 40, 20, 4), (80, 20, 3, 1), (50, 50, 6, 2), (36, 14, 40, 8), (256, 256, 2, 1), (2, 2, 7, 3), (511, 2, 2, 1), (17, 16, 9, 2),
                                              (512, 6, 1, 1), (512, 512, 1, 2), (64, 64, 1, 0), (24, 10, 100, 3)])
def test_many_tokens_of_every_form(type, interleaved, head, rotary, H, HK):
    """From 2368 tokens on a B200 a CTA has one to four of them and 128 or 256 threads, by what keeps them busy; 2603 is a multiple of neither two, three nor four."""
    from amdgpu_rustdsl_b200 import Rope, rope_rotate
    rope = Rope(rotary, interleaved=interleaved, scaling={"kind": "yarn", "factor": 4.0, "original": 4096})
    B, S = 19, 137
    x, y = R.make(B, S, H, head, R.TYPES[type]), R.make(B, S, HK, head, R.TYPES[type], 1)
    positions = torch.randint(0, 1 << 20, (B, S), generator=torch.Generator().manual_seed(2)).cuda()
    out, y_out = torch.full_like(x, math.nan), torch.full_like(y, math.nan)
    rope_rotate(rope, x, positions, out, y=y, y_out=y_out)
    R.check(rope, x, positions, out)
    R.check(rope, y, positions, y_out)
    back, y_back = out.clone(), y_out.clone()
    rope_rotate(rope, back, positions, y=y_back, backward=True)
    R.check(rope, out, positions, back, True)
    R.check(rope, y_out, positions, y_back, True)
