"""Python entry of rotary positions: queries and keys are turned by their tokens' positions on their way to the attention or a cache.

    rope = Rope(128, base=500000.0, scaling={"kind": "yarn", "factor": 4.0, "original": 8192}, device=dev)   # once
    rope_rotate(rope, q, positions, y=k)                                                                       # per layer, in place
    rope_rotate(rope, grad_q, positions, y=grad_k, backward=True)                                              # its gradient

PyTorch owns memory and streams only; the call goes to the sm_100a kernels behind the C ABI of ``include/fmha_rope_abi.h``, runs on torch's current stream of x's device (or
``stream``, a raw handle) and does not wait for it. Wrong arguments raise ``ValueError``.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from fractions import Fraction

from . import _abi
from .kv4 import _check, _errors
from .ops import _raw_stream

# 2 pi to 40 digits, of which 64-bit phases need 20
_TWO_PI = Fraction(62831853071795864769252867665590057683943, 10 ** 40)
MAX_HEAD_DIM = 512
_NO_ROWS, _NO_STRIDES = (0,) * 8, (0,) * 4
_ARGS = struct.Struct("@20q10If4x").pack
assert struct.calcsize("@20q10If4x") == C.sizeof(_abi.RopeArgs)
_kinds, _entry = {}, None


def _types(torch):
    if not _kinds:
        _kinds.update({torch.bfloat16: 0, torch.float16: 1, torch.float32: 2})
    return _kinds


def _load():
    """The C entry with its arguments as bytes."""
    global _entry
    entry = _abi.load()["fmha_rope_rotate"]
    entry.restype, entry.argtypes = C.c_int, [C.c_char_p, C.c_void_p, C.c_char_p, C.c_size_t]
    _entry = entry
    return entry


def _number(who, scaling, name, default=None):
    value = scaling.get(name, default)
    if not isinstance(value, (int, float)) or not math.isfinite(value) or value <= 0:
        raise ValueError(f"Rope: scaling {who!r} needs a positive number {name!r}")
    return float(value)


def rope_frequencies(rotary, base=10000.0, scaling=None):
    """(radians per position of the ``rotary`` / 2 pairs, what the results are multiplied by), in Python's 64 bits.

    Pair i turns by base^(-2 i / rotary) a position. ``scaling`` stretches that for contexts longer than the one that a model was trained on, by ``factor``:
      {"kind": "linear", "factor"}    all frequencies / factor
      {"kind": "ntk", "factor"}       the base grows to base * factor^(rotary / (rotary - 2)): the fastest pair stays, the slowest is / factor
      {"kind": "yarn", "factor", "original", "fast" (32), "slow" (1), "attention"}
                                      pairs that turn more than ``fast`` times in the ``original`` context stay, those below ``slow`` turns are / factor, with a ramp over the pairs
                                      between; results times 0.1 ln factor + 1, or ``attention`` where given
      {"kind": "bands", "factor", "original", "low" (1), "high" (4)}
                                      by wavelength: below original / high as they are, above original / low divided, between the two blended
    """
    if not isinstance(rotary, int) or rotary < 2 or rotary % 2 or rotary > MAX_HEAD_DIM:
        raise ValueError(f"Rope: rotary must be an even number from 2 to {MAX_HEAD_DIM}, not {rotary}")
    if not isinstance(base, (int, float)) or not math.isfinite(base) or base < 1.0:
        raise ValueError("Rope: base must be a number from 1 on")
    n, attention = rotary // 2, 1.0
    f = [float(base) ** (-i / n) for i in range(n)]
    if scaling is None:
        return f, attention
    kind, known = scaling.get("kind"), {"linear": (), "ntk": (), "yarn": ("original", "fast", "slow", "attention"), "bands": ("original", "low", "high")}
    if kind not in known or set(scaling) - {"kind", "factor", *known[kind]}:
        raise ValueError(f"Rope: scaling must be one of {sorted(known)} with its own numbers, not {dict(scaling)}")
    factor = _number(kind, scaling, "factor")
    if kind == "linear":
        return [x / factor for x in f], attention
    if kind == "ntk":
        return (f if n == 1 else [(base * factor ** (n / (n - 1))) ** (-i / n) for i in range(n)]), attention
    original = _number(kind, scaling, "original")
    if kind == "yarn":
        fast, slow = _number(kind, scaling, "fast", 32.0), _number(kind, scaling, "slow", 1.0)
        if fast < slow or base <= 1.0:
            raise ValueError("Rope: scaling 'yarn' needs fast not below slow and a base above 1")
        # the pair that turns so many times in the original context
        at = [rotary * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (fast, slow)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary - 1)
        ramp = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(n)]
        attention = _number(kind, scaling, "attention", 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0)
        return [x / factor * r + x * (1.0 - r) for x, r in zip(f, ramp)], attention
    low, high = _number(kind, scaling, "low", 1.0), _number(kind, scaling, "high", 4.0)
    if high <= low:
        raise ValueError("Rope: scaling 'bands' needs high above low")
    smooth = [min(max((original * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for x in f]
    return [(1.0 - s) * x / factor + s * x for x, s in zip(f, smooth)], attention


class Rope:
    """The frequencies of rotary positions on a device, as fractions of a turn in 64-bit fixed point: angles of positions of any 32-bit size are exact to 2^-33 of a turn.

    rotary       elements of a head that are turned, its first ones (an even number up to 512)
    interleaved  neighbours (2 i, 2 i + 1) are a pair; else (i, rotary / 2 + i)
    base, scaling  as in ``rope_frequencies``; or ``frequencies``, radians per position of each pair from 0 on, and ``factor``, what results are multiplied by
    """
    __slots__ = ("rotary", "interleaved", "factor", "frequencies", "turns", "address", "device", "index")

    def __init__(self, rotary, *, base=10000.0, interleaved=False, scaling=None, frequencies=None, factor=None, device="cuda"):
        import torch
        computed, attention = rope_frequencies(rotary, base, scaling)
        if frequencies is not None:
            if scaling is not None:
                raise ValueError("Rope: frequencies or scaling, not both")
            computed = [float(x) for x in frequencies]
            if len(computed) != rotary // 2 or not all(math.isfinite(x) and x >= 0.0 for x in computed):
                raise ValueError(f"Rope: frequencies must be {rotary // 2} numbers from 0 on")
        factor = attention if factor is None else float(factor)
        if not 0.0 < factor < 3.0e38:
            raise ValueError("Rope: factor must be a positive number")
        self.rotary, self.interleaved, self.factor, self.frequencies = rotary, bool(interleaved), factor, tuple(computed)
        # a turn is 2^64; whole turns (and with them the highest bit's sign) fall out
        turns = [round(Fraction(x) / _TWO_PI * 2 ** 64) % 2 ** 64 for x in computed]
        self.turns = torch.tensor([x - 2 ** 64 if x >= 2 ** 63 else x for x in turns], dtype=torch.int64).to(device)
        self.address, self.device, self.index = self.turns.data_ptr(), self.turns.device, self.turns.get_device()


def _rope_rows(name, x, rope, like):
    """(address, strides) of x, [B, S, heads, head size] of like's type and sizes but for the heads."""
    shape, other, (sb, ss, sh, sd) = x.shape, like.shape, x.stride()
    if x.dtype != like.dtype or shape[:2] != other[:2] or shape[3] != other[3]:
        raise ValueError(f"rope_rotate: {name} must have x's type, sequences, rows and head size")
    if x.get_device() != rope.index or (sd != 1 and shape[3] > 1):
        raise ValueError(f"rope_rotate: {name} must be on the Rope's device, its last dimension dense")
    return x.data_ptr(), sb, ss, sh


def rope_rotate(rope, x, positions, out=None, *, y=None, y_out=None, backward=False, stream=None):
    """Turns the rows of x, and of y, by their tokens' positions: x [B, S, heads, head size] bf16, f16 or f32 (strided), y the same with heads of its own number (queries and keys).

    positions  int32 or int64 [B, S] (strided; ``expand`` is fine), any numbers, negative ones too
    out, y_out where the results go, else in place. An output is its input or shares no memory with it, nor with the other's input or output (heads of the same rows do not)
    backward   the transposed matrix: x is the gradient of the results, and out becomes the gradient of what went in
    """
    import torch
    dtype, shape, index = x.dtype, x.shape, rope.index
    kind = _types(torch).get(dtype)
    if kind is None:
        raise ValueError(f"rope_rotate: x must be bf16, f16 or f32, not {dtype}")
    if len(shape) != 4 or not rope.rotary <= shape[3] <= MAX_HEAD_DIM:
        raise ValueError(f"rope_rotate: x must be [B, S, heads, {rope.rotary} to {MAX_HEAD_DIM}], not {tuple(shape)}")
    B, S, H, head = shape
    rows = _rope_rows("x", x, rope, x)
    rows_out, heads_y, more = rows, 0, _NO_ROWS
    if out is None:
        out = x
    elif out is not x:
        sb, ss, sh, sd = out.stride() if out.shape == shape else _NO_STRIDES
        if sd == 1 and out.dtype == dtype and out.get_device() == index:   # (as a rule, and the quickest way to know)
            rows_out = out.data_ptr(), sb, ss, sh
        else:
            if out.dim() != 4 or out.shape[2] != H:
                raise ValueError("rope_rotate: out must have x's heads")
            rows_out = _rope_rows("out", out, rope, x)
    if y is not None:
        shape_y = y.shape
        if len(shape_y) != 4:
            raise ValueError("rope_rotate: y must have x's type, sequences, rows and head size")
        heads_y, first = shape_y[2], _rope_rows("y", y, rope, x)
        if y_out is None or y_out is y:
            more = first + first
        else:
            sb, ss, sh, sd = y_out.stride() if y_out.shape == shape_y else _NO_STRIDES
            if sd == 1 and y_out.dtype == dtype and y_out.get_device() == index:
                more = first + (y_out.data_ptr(), sb, ss, sh)
            else:
                if y_out.dim() != 4 or y_out.shape[2] != heads_y:
                    raise ValueError("rope_rotate: y_out must have y's heads")
                more = first + _rope_rows("y_out", y_out, rope, x)
    elif y_out is not None:
        raise ValueError("rope_rotate: y_out without y")
    wide = positions.dtype == torch.int64
    if not (wide or positions.dtype == torch.int32) or positions.shape != (B, S) or positions.get_device() != index:
        raise ValueError(f"rope_rotate: positions must be int32 or int64 of shape {(B, S)} on the Rope's device")
    tokens = B * S
    if tokens > 1 << 30 or H > 1 << 30 or heads_y > 1 << 30:   # (here, in numbers of any size: the struct's have 32 bits)
        raise ValueError("rope_rotate: more than 2^30 tokens or heads")
    if tokens == 0 or H + heads_y == 0:
        return out
    if H == 0:   # only y has heads
        rows, rows_out, more, H, heads_y = more[:4], more[4:], _NO_ROWS, heads_y, 0
    if index < 0:
        raise ValueError("rope_rotate: the Rope must be on a CUDA device")
    # fmha_rope_args, as bytes: an eighth of the time that setting the fields one by one takes
    args = _ARGS(*rows, *rows_out, *more, rope.address, positions.data_ptr(), *positions.stride(), wide, B, S, H, heads_y, head, rope.rotary, kind, rope.interleaved, bool(backward), rope.factor)
    raw = stream if stream is not None else _raw_stream(torch, rope.device)
    rotate = _entry or _load()
    if torch.cuda.current_device() == index:
        rc = rotate(args, raw, _errors.text, 256)
    else:
        with torch.cuda.device(rope.device):
            rc = rotate(args, raw, _errors.text, 256)
    if rc:
        _check("rope_rotate", rc)
    return out
