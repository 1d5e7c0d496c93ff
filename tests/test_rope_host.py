"""Rotary positions without a GPU: frequencies, fixed point, and that wrong arguments are refused with a message before anything is launched or read."""
import ctypes as C
import math

import pytest
import torch

FAKE = 1 << 24   # an aligned address that nothing follows: every call here is refused


def test_frequencies_fall_from_one_and_are_stretched_as_they_say():
    from amdgpu_rustdsl_b200 import rope_frequencies
    f, factor = rope_frequencies(128)
    assert factor == 1.0 and len(f) == 64 and f[0] == 1.0 and math.isclose(f[63], 10000.0 ** (-126 / 128), rel_tol=1e-15)
    assert rope_frequencies(128, scaling={"kind": "linear", "factor": 4})[0] == [x / 4 for x in f]
    ntk = rope_frequencies(128, scaling={"kind": "ntk", "factor": 4})[0]
    assert ntk[0] == 1.0 and math.isclose(ntk[63], f[63] / 4, rel_tol=1e-13) and rope_frequencies(2, scaling={"kind": "ntk", "factor": 4})[0] == [1.0]
    yarn, factor = rope_frequencies(128, scaling={"kind": "yarn", "factor": 4, "original": 4096})
    turns = [4096 * x / (2 * math.pi) for x in f]
    assert all(a == b for a, b, t in zip(yarn, f, turns) if t > 40) and all(math.isclose(a, b / 4, rel_tol=1e-14) for a, b, t in zip(yarn, f, turns) if t < 0.8)
    assert all(b / 4 - 1e-18 <= a <= b for a, b in zip(yarn, f)) and math.isclose(factor, 0.1 * math.log(4) + 1)
    assert rope_frequencies(128, scaling={"kind": "yarn", "factor": 4, "original": 4096, "attention": 1.5})[1] == 1.5
    bands, factor = rope_frequencies(128, 500000.0, {"kind": "bands", "factor": 8, "original": 8192})
    f = rope_frequencies(128, 500000.0)[0]
    wavelengths = [2 * math.pi / x for x in f]
    assert factor == 1.0 and all(a == b for a, b, w in zip(bands, f, wavelengths) if w < 2048) and all(a == b / 8 for a, b, w in zip(bands, f, wavelengths) if w > 8192)
    assert all(b / 8 <= a <= b for a, b in zip(bands, f))


def test_fixed_point_is_the_frequency_in_turns():
    from amdgpu_rustdsl_b200 import Rope
    rope = Rope(4, frequencies=[2 * math.pi, 1.0], device="cpu")
    # 2 pi as a double is 2.4e-16 below 2 pi: as good as a whole turn, which is nothing
    assert abs(int(rope.turns[0])) <= 2 ** 64 * 5e-17 and abs(int(rope.turns[1]) - 2 ** 64 / (2 * math.pi)) < 2 ** 13
    assert Rope(4, frequencies=[5.0, 0.0], device="cpu").turns[0] < 0   # more than half a turn


@pytest.mark.parametrize("call", [dict(rotary=3), dict(rotary=0), dict(rotary=514), dict(rotary=8.0), dict(rotary=8, base=0.5), dict(rotary=8, base=math.nan), dict(rotary=8, scaling={"kind": "other", "factor": 2}),
                                  dict(rotary=8, scaling={"kind": "linear"}), dict(rotary=8, scaling={"kind": "linear", "factor": -1}), dict(rotary=8, scaling={"kind": "linear", "factor": 2, "original": 5}),
                                  dict(rotary=8, scaling={"kind": "yarn", "factor": 2}), dict(rotary=8, scaling={"kind": "yarn", "factor": 2, "original": 10, "fast": 1, "slow": 2}),
                                  dict(rotary=8, scaling={"kind": "bands", "factor": 2, "original": 10, "low": 4, "high": 4}), dict(rotary=8, frequencies=[1.0]), dict(rotary=4, frequencies=[1.0, -1.0]),
                                  dict(rotary=4, frequencies=[1.0, math.inf]), dict(rotary=4, frequencies=[1.0, 1.0], scaling={"kind": "linear", "factor": 2}), dict(rotary=8, factor=0.0), dict(rotary=8, factor=math.inf)])
def test_bad_frequencies_are_refused(call):
    from amdgpu_rustdsl_b200 import Rope
    with pytest.raises(ValueError, match="Rope"):
        Rope(device="cpu", **call)


def _args(abi, **change):
    """Queries of 4 and keys of 2 heads of 64, packed, into memory of their own."""
    rows = lambda at, heads: abi.Kv4Rows(at, 3 * heads * 64, heads * 64, 64)
    a = abi.RopeArgs(x=rows(FAKE, 4), x_out=rows(2 * FAKE, 4), y=rows(3 * FAKE, 2), y_out=rows(4 * FAKE, 2), turns=FAKE, positions=FAKE, positions_stride_b=3, positions_stride_s=1,
                     B=2, S=3, heads_x=4, heads_y=2, head_dim=64, rotary=64, factor=1.0)
    for k, v in change.items():
        setattr(a, k, v)
    return a


def _refused(abi, message, **change):
    err = C.create_string_buffer(256)
    assert abi.load().fmha_rope_rotate(_args(abi, **change), None, err, 256) == 6 and message in err.value.decode(), err.value


@pytest.mark.parametrize("change,message", [
    ({"type": 3}, "bf16"), ({"head_dim": 0}, "heads have"), ({"head_dim": 1024}, "heads have"), ({"rotary": 0}, "heads have"), ({"rotary": 63}, "heads have"), ({"rotary": 66}, "heads have"),
    ({"factor": 0.0}, "factor"), ({"factor": math.nan}, "factor"), ({"heads_x": 0}, "no heads"), ({"turns": None}, "turns"), ({"turns": FAKE + 4}, "turns"), ({"positions": None}, "positions"),
    ({"positions": FAKE + 2}, "positions"), ({"positions": FAKE + 4, "positions_64": 1}, "positions"), ({"B": 1 << 20, "S": 1 << 11}, "2^30")])
def test_bad_calls_are_refused(abi, change, message):
    _refused(abi, message, **change)


def test_bad_rows_are_refused(abi):
    rows = abi.Kv4Rows
    for name in ("x", "x_out", "y", "y_out"):
        _refused(abi, "must be given", **{name: rows(None, 512, 128, 64)})
        _refused(abi, "aligned", **{name: rows(FAKE + 1, 512, 128, 64)})
        _refused(abi, "negative", **{name: rows(5 * FAKE, 512, -128, 64)})
        _refused(abi, "larger than any memory", **{name: rows(5 * FAKE, 1 << 60, 128, 64)})
    _refused(abi, "aligned", type=2, x=rows(FAKE + 2, 768, 256, 64))
    # outputs that write an element twice
    for strides in ((0, 256, 64), (768, 0, 64), (768, 256, 0), (768, 256, 63), (767, 256, 64), (768, 255, 64)):
        _refused(abi, "share memory", x_out=rows(2 * FAKE, *strides))
    # outputs on inputs, but not their elements
    _refused(abi, "x_out must be x", x_out=rows(FAKE + 2, 768, 256, 64))
    _refused(abi, "x_out must be x", x_out=rows(FAKE, 768, 256, 64 + 0), x=rows(FAKE, 1536, 256, 64))
    _refused(abi, "y_out must be y", y_out=rows(3 * FAKE + 128, 384, 128, 64))
    _refused(abi, "other input or output", y_out=rows(2 * FAKE, 384, 128, 64))
    _refused(abi, "other input or output", y_out=rows(FAKE, 384, 128, 64))
    _refused(abi, "other input or output", y=rows(2 * FAKE + 512, 384, 128, 64))


def test_nothing_to_do_is_no_error(abi):
    err = C.create_string_buffer(256)
    for change in ({"B": 0}, {"S": 0}):
        assert abi.load().fmha_rope_rotate(_args(abi, **change), None, err, 256) == 0
    assert abi.load().fmha_rope_rotate(None, None, err, 256) == 6


def test_the_python_entry_refuses_on_the_cpu():
    from amdgpu_rustdsl_b200 import Rope, rope_rotate
    rope = Rope(8, device="cpu")
    x, at = torch.zeros(2, 3, 4, 16, dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int32)
    for call, message in ((lambda: rope_rotate(rope, x.double(), at), "bf16"), (lambda: rope_rotate(rope, x[..., :6], at), "x must be"), (lambda: rope_rotate(rope, x[0], at), "x must be"),
                          (lambda: rope_rotate(rope, x.transpose(2, 3).contiguous().transpose(2, 3), at), "dense"), (lambda: rope_rotate(rope, x, at, x[:, :, :2]), "heads"),
                          (lambda: rope_rotate(rope, x, at, x.float()), "type"), (lambda: rope_rotate(rope, x, at, y=x[:1]), "sequences"), (lambda: rope_rotate(rope, x, at, y=x, y_out=x[:, :, :1]), "heads"),
                          (lambda: rope_rotate(rope, x, at, y_out=x), "without y"), (lambda: rope_rotate(rope, x, at.float()), "positions"), (lambda: rope_rotate(rope, x, at[:, :2]), "positions")):
        with pytest.raises(ValueError, match=message):
            call()
    assert rope_rotate(rope, x[:, :0], at[:, :0]).shape == (2, 0, 4, 16)
