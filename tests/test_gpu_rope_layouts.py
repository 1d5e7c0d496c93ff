"""Queries and keys that lie between one another without sharing an element, against the same rotated apart."""
import pytest
import torch

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
