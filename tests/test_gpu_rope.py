"""Rotary positions on the GPU, against the formula in 64 bits and its differences.

Tolerances, per pair (a, b) with results a', b': the phase is off by 2^-33 of a turn at most and its quarter's rest is f32 (2^-27 of half a turn), sine and cosine come out within 2 units in the
last place, two products and a sum in f32: together below 16 * 2^-24 (|a| + |b|) factor. Then one rounding to the type, half a step of the result or of its smallest one."""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def turned(rope, x, positions, backward=False):
    """The formula in 64 bits, and |a| + |b| of each element's pair (0 where nothing is turned)."""
    n = rope.rotary // 2
    x, size = x.double().cpu(), torch.zeros(x.shape, dtype=torch.float64)
    f = torch.tensor(rope.frequencies, dtype=torch.float64)
    angle = (positions.cpu().double()[..., None] * f)[:, :, None]
    cos, sin = torch.cos(angle) * rope.factor, torch.sin(angle) * rope.factor * (-1 if backward else 1)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if rope.interleaved else (slice(0, n), slice(n, 2 * n))
    a, b, out = x[..., first], x[..., second], x.clone()
    out[..., first], out[..., second] = a * cos - b * sin, a * sin + b * cos
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return out, size * rope.factor


def check(rope, x, positions, got, backward=False):
    want, size = turned(rope, x, positions, backward)
    info = torch.finfo(x.dtype)
    step = torch.maximum(want.abs() * info.eps / 2, torch.tensor(info.tiny * info.eps / 2, dtype=torch.float64))
    room = torch.where(size > 0, (16 * 2.0 ** -24) * size * (1 + info.eps) + step, 0.0)
    assert ((got.cpu().double() - want).abs() <= room).all(), ((got.cpu().double() - want).abs() - room).max()


def make(B, S, H, head, dtype, seed=0):
    return torch.randn(B, S, H, head, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("head,rotary", [(128, 128), (128, 64), (96, 40), (64, 64), (80, 20), (50, 50), (36, 14), (256, 256), (2, 2), (512, 512), (511, 2), (17, 16), (512, 6)])
def test_heads_and_parts_of_all_sizes(type, interleaved, head, rotary):
    from amdgpu_rustdsl_b200 import Rope, rope_rotate
    rope = Rope(rotary, interleaved=interleaved)
    x, y = make(2, 7, 5, head, TYPES[type]), make(2, 7, 2, head, TYPES[type], 1)
    positions = torch.randint(0, 1 << 17, (2, 7), dtype=torch.int32, generator=torch.Generator().manual_seed(2)).cuda()
    for backward in (False, True):
        out, y_out = torch.full_like(x, math.nan), torch.full_like(y, math.nan)
        assert rope_rotate(rope, x, positions, out, y=y, y_out=y_out, backward=backward) is out
        check(rope, x, positions, out, backward)
        check(rope, y, positions, y_out, backward)
        within, y_within = x.clone(), y.clone()
        rope_rotate(rope, within, positions, y=y_within, backward=backward)
        assert torch.equal(within, out) and torch.equal(y_within, y_out)


@pytest.mark.parametrize("B,S,H,HK", [(1, 1, 1, 0), (1, 1, 40, 8), (64, 1, 32, 8), (3, 333, 12, 4), (1, 4097, 8, 1), (2, 2500, 1, 1), (300, 1, 64, 8), (1, 1, 0, 3)])
def test_numbers_of_tokens_and_heads(B, S, H, HK):
    from amdgpu_rustdsl_b200 import Rope, rope_rotate
    rope = Rope(128, base=500000.0, scaling={"kind": "yarn", "factor": 8.0, "original": 4096})
    x, y = make(B, S, H, 128, torch.bfloat16), make(B, S, HK, 128, torch.bfloat16, 1)
    positions = (torch.arange(S) + torch.arange(B)[:, None] * 1000).int().cuda()
    out, y_out = torch.full_like(x, math.nan), torch.full_like(y, math.nan)
    rope_rotate(rope, x, positions, out, y=y if HK else None, y_out=y_out if HK else None)
    check(rope, x, positions, out)
    check(rope, y, positions, y_out)


@pytest.mark.parametrize("type", ["bf16", "f32"])
def test_slices_of_a_projection_views_and_odd_alignment(type):
    """Queries and keys as heads of one row, in place and out of it; heads in front of tokens; rows that start off the wide accesses' boundaries; one row for all (stride 0)."""
    from amdgpu_rustdsl_b200 import Rope, rope_rotate
    rope, dtype = Rope(64), TYPES[type]
    positions = torch.randint(0, 9000, (3, 5), dtype=torch.int64, generator=torch.Generator().manual_seed(4)).cuda()
    for shift, pad in itertools.product((0, 1, 2, 4), (0, 1, 6)):
        row = 8 * 96 + pad
        flat = torch.randn(3 * 5 * row + 8, generator=torch.Generator().manual_seed(shift)).to(dtype).cuda()
        qkv = flat[shift:shift + 15 * row].view(3, 5, row)[..., :8 * 96].unflatten(-1, (8, 96))
        before = flat.clone()
        q, k = qkv[:, :, :4], qkv[:, :, 4:6]
        x, y = q.clone(), k.clone()
        q_out, k_out = torch.empty_like(x), torch.empty_like(y)
        rope_rotate(rope, q, positions, q_out, y=k, y_out=k_out)
        assert torch.equal(flat, before)
        check(rope, x, positions, q_out)
        check(rope, y, positions, k_out)
        rope_rotate(rope, q, positions, y=k)
        assert torch.equal(q, q_out) and torch.equal(k, k_out)
        after = before.clone()
        after[shift:shift + 15 * row].view(3, 5, row)[..., :6 * 96] = torch.cat([q_out, k_out], 2).flatten(2)
        assert torch.equal(flat, after)   # values, padding and what is around are as they were
    x = make(3, 5, 6, 96, dtype)
    good = rope_rotate(rope, x, positions, torch.empty_like(x))
    heads_first = torch.empty(3, 6, 5, 96, dtype=dtype, device="cuda").transpose(1, 2)
    rope_rotate(rope, x.transpose(1, 2).contiguous().transpose(1, 2), positions, heads_first)
    assert torch.equal(heads_first, good)
    one = x[:1, :1, :1].expand(3, 5, 6, 96)
    out = rope_rotate(rope, one, positions, torch.empty_like(x))
    check(rope, one, positions, out)
    same = positions[:1].expand(3, 5)
    check(rope, x, same, rope_rotate(rope, x, same, torch.empty_like(x)))
    check(rope, x, positions.t().contiguous().t(), rope_rotate(rope, x, positions.t().contiguous().t(), torch.empty_like(x)))


def test_positions_of_any_size():
    """32-bit positions far out, negative ones, 64-bit ones: the angles are exact to 2^-33 of a turn for 32 bits (frequencies are held to 2^-65 of a turn)."""
    from fractions import Fraction
    from amdgpu_rustdsl_b200 import Rope, rope_rotate
    rope = Rope(32, base=10000.0)
    at = torch.tensor([[0, 1, -1, 131071, -131072, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31]])
    x = torch.zeros(1, 8, 1, 32, device="cuda")
    x[..., :16] = 1.0
    two_pi = Fraction(62831853071795864769252867665590057683943, 10 ** 40)
    want = torch.zeros(8, 32, dtype=torch.float64)
    for s, p in enumerate(at[0].tolist()):
        for i, f in enumerate(rope.frequencies):
            turns = Fraction(f) * p / two_pi
            part = float((turns - round(turns)) * two_pi)
            want[s, i], want[s, 16 + i] = math.cos(part), math.sin(part)
    for positions in (at.int().cuda(), at.cuda()):
        out = rope_rotate(rope, x, positions, torch.empty_like(x))
        assert ((out[0, :, 0].cpu().double() - want).abs() <= 16 * 2.0 ** -24 + 2.0 ** -31).all()
    # a turn later by a 64-bit position: frequency of 2^-40 turns
    slow = Rope(2, frequencies=[2 * math.pi * 2.0 ** -40])
    y = torch.tensor([1.0, 0.0], device="cuda").view(1, 1, 1, 2)
    out = rope_rotate(slow, y, torch.tensor([[2 ** 40 + 2 ** 38]], device="cuda"), torch.empty_like(y))
    assert (out.flatten().cpu() - torch.tensor([0.0, 1.0])).abs().max() < 2.0 ** -20


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("scaling", [None, {"kind": "yarn", "factor": 4.0, "original": 2048}])
def test_gradient_against_the_formula_and_differences(interleaved, scaling):
    """The gradient of sum(w * rope(x)) is rope backward of w; rope backward undoes rope, times the factor's square."""
    from amdgpu_rustdsl_b200 import Rope, rope_rotate
    rope = Rope(24, interleaved=interleaved, scaling=scaling)
    x, w = make(2, 3, 2, 32, torch.float32, 5), make(2, 3, 2, 32, torch.float32, 6)
    positions = torch.tensor([[5, 900, 3], [0, 77777, 12]], dtype=torch.int32, device="cuda")
    grad = rope_rotate(rope, w, positions, torch.empty_like(w), backward=True)
    leaf = x.double().cpu().requires_grad_()
    n, f = 12, torch.tensor(rope.frequencies, dtype=torch.float64)
    angle = (positions.cpu().double()[..., None] * f)[:, :, None]
    first, second = (slice(0, 24, 2), slice(1, 24, 2)) if interleaved else (slice(0, n), slice(n, 24))
    a, b = leaf[..., first], leaf[..., second]
    g = w.double().cpu()
    loss = rope.factor * ((a * angle.cos() - b * angle.sin()) * g[..., first] + (a * angle.sin() + b * angle.cos()) * g[..., second]).sum() + (leaf[..., 24:] * g[..., 24:]).sum()
    loss.backward()
    assert (grad.cpu().double() - leaf.grad).abs().max() <= 16 * 2.0 ** -24 * 2 * w.abs().max().item() * rope.factor
    # differences: the map is linear, so that a difference of any size is exact but for rounding
    for e in range(0, 32, 5):
        step = torch.zeros_like(x)
        step[0, 1, 1, e] = 1.0
        high, low = (rope_rotate(rope, x + s * step, positions, torch.empty_like(x)).double() for s in (1.0, -1.0))
        slope = ((high - low) / 2 * w.double()).sum().item()
        assert abs(slope - grad[0, 1, 1, e].item()) <= 1e-4
    back = rope_rotate(rope, rope_rotate(rope, x, positions, torch.empty_like(x)), positions, torch.empty_like(x), backward=True)
    again = torch.cat([x[..., :24] * rope.factor ** 2, x[..., 24:]], -1)
    assert (back - again).abs().max() <= 64 * 2.0 ** -24 * 2 * x.abs().max().item() * rope.factor ** 2


def test_infinities_and_nan_stay_in_their_pairs():
    from amdgpu_rustdsl_b200 import Rope, rope_rotate
    rope, positions = Rope(64), torch.full((1, 4), 3, dtype=torch.int32, device="cuda")
    x = make(1, 4, 3, 128, torch.bfloat16)
    good = rope_rotate(rope, x, positions, torch.empty_like(x))
    x[0, 1, 1, 5], x[0, 2, 0, 40], x[0, 3, 2, 100] = math.inf, math.nan, math.nan
    out = rope_rotate(rope, x, positions, torch.empty_like(x))
    touched = torch.zeros_like(x, dtype=torch.bool)
    touched[0, 1, 1, [5, 37]] = touched[0, 2, 0, [8, 40]] = touched[0, 3, 2, 100] = True
    assert not torch.isfinite(out[touched].float()).any() and torch.equal(out[~touched], good[~touched])


def test_other_streams_and_graphs():
    from amdgpu_rustdsl_b200 import Rope, rope_rotate
    rope = Rope(128)
    x, positions = make(2, 100, 8, 128, torch.bfloat16), torch.arange(200, dtype=torch.int32, device="cuda").view(2, 100)
    good = rope_rotate(rope, x, positions, torch.empty_like(x))
    torch.cuda.synchronize()
    side, late, out = torch.cuda.Stream(), torch.zeros_like(x), torch.empty_like(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        late.copy_(x)
        rope_rotate(rope, late, positions, out)
    side.synchronize()
    assert torch.equal(out, good)
    out.zero_()
    torch.cuda.synchronize()
    rope_rotate(rope, x, positions, out, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, good)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rope_rotate(rope, x, positions, out)
    positions += 5
    graph.replay()
    torch.cuda.synchronize()
    check(rope, x, positions, out)


def test_more_than_32_bits_of_bytes():
    from amdgpu_rustdsl_b200 import Rope, rope_rotate
    rope, stride = Rope(128), (5 << 30) // 2
    flat = torch.empty(stride + 256, dtype=torch.bfloat16, device="cuda")
    x = flat.as_strided((2, 1, 2, 128), (stride, 256, 128, 1))
    x.copy_(make(2, 1, 2, 128, torch.bfloat16))
    positions = torch.tensor([[7], [8]], dtype=torch.int32, device="cuda")
    before = x.clone()
    rope_rotate(rope, x, positions)
    check(rope, before, positions, x)


def test_refusals_of_the_python_entry():
    from amdgpu_rustdsl_b200 import Rope, rope_rotate
    rope = Rope(64)
    x, positions = make(2, 3, 4, 64, torch.bfloat16), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for call, message in ((lambda: rope_rotate(rope, x.cpu(), positions), "device"), (lambda: rope_rotate(rope, x, positions.cpu()), "device"), (lambda: rope_rotate(rope, x[:, :, :, :32], positions), "x must be"),
                          (lambda: rope_rotate(rope, x[:1, :1, :1].expand(2, 3, 4, 64), positions), "share memory"), (lambda: rope_rotate(rope, x[:, :, :3], positions, x[:, :, 1:]), "x_out must be x"),
                          (lambda: rope_rotate(rope, x, positions, torch.empty_like(x), y=x, y_out=x), "other input"), (lambda: rope_rotate(rope, x[:, :, :2], positions, y=x[:, :, 1:]), "other input")):
        with pytest.raises(ValueError, match=message):
            call()
