"""The 4-bit cache's C ABI without a GPU: exports, and that wrong arguments are refused with a message before anything is launched or read."""
import ctypes as C
import os
import re

import pytest
import torch

from tests import kv4_reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 1 << 20   # an aligned address that nothing follows: every call here is refused


def test_every_declared_symbol_is_exported(abi):
    declared = set(re.findall(r"\b(fmha_kv4_[a-z0-9_]+)\s*\(", open(os.path.join(ROOT, "include", "fmha_kv4_abi.h")).read()))
    assert declared == set(abi.KV4_EXPORTS)
    for name in declared:
        assert getattr(abi.load(), name) is not None


def _cache(abi, **change):
    c = abi.Kv4CacheArgs(pool=FAKE, table=FAKE, lengths=FAKE, pages=8, B=2, HK=2, page=64, table_width=4)
    for k, v in change.items():
        setattr(c, k, v)
    return c


def _rows(abi, **change):
    r = abi.Kv4Rows(FAKE, 2 * 3 * 128, 2 * 128, 128)
    for k, v in change.items():
        setattr(r, k, v)
    return r


BAD_CACHES = [({"pool": None}, "must be given"), ({"table": None}, "must be given"), ({"lengths": None}, "must be given"), ({"pool": FAKE + 8}, "16-byte aligned"),
              ({"page": 48}, "16, 32, 64 or 128"), ({"page": 0}, "16, 32, 64 or 128"), ({"page": 256}, "16, 32, 64 or 128"), ({"B": 0}, "no sequences"), ({"HK": 0}, "no sequences"),
              ({"pages": 0}, "no sequences"), ({"table_width": 0}, "no sequences"), ({"pages": 1 << 31}, "2^31"), ({"table_width": 1 << 26}, "2^31"),
              ({"B": 1 << 16, "HK": 1 << 15}, "2^30")]


@pytest.mark.parametrize("change,message", BAD_CACHES)
def test_bad_caches_are_refused(abi, change, message):
    lib, err = abi.load(), C.create_string_buffer(256)
    rows = _rows(abi)
    assert lib.fmha_kv4_append(_cache(abi, **change), rows, rows, 3, None, None, err, 256) == 6 and message in err.value.decode()
    assert lib.fmha_kv4_read(_cache(abi, **change), rows, rows, 3, 0, None, None, err, 256) == 6 and message in err.value.decode()
    assert lib.fmha_kv4_attend(_cache(abi, **change), abi.Kv4AttendArgs(q=rows, out=FAKE, S=3, H=2, scale=1.0), None, err, 256) == 6 and message in err.value.decode()
    assert lib.fmha_kv4_attend_workspace(_cache(abi, **change), abi.Kv4AttendArgs(q=rows, out=FAKE, S=3, H=2, scale=1.0)) == 0


@pytest.mark.parametrize("change", [{"data": None}, {"data": FAKE + 2}, {"stride_b": 4}, {"stride_s": 129}, {"stride_h": 3}])
def test_bad_rows_are_refused(abi, change):
    lib, err = abi.load(), C.create_string_buffer(256)
    good, bad = _rows(abi), _rows(abi, **change)
    assert lib.fmha_kv4_append(_cache(abi), bad, good, 3, None, None, err, 256) == 6 and "k" in err.value.decode()
    assert lib.fmha_kv4_append(_cache(abi), good, bad, 3, None, None, err, 256) == 6 and "v" in err.value.decode()
    assert lib.fmha_kv4_read(_cache(abi), good, bad, 3, 1, None, None, err, 256) == 6
    assert lib.fmha_kv4_attend(_cache(abi), abi.Kv4AttendArgs(q=bad, out=FAKE, S=3, H=2, scale=1.0), None, err, 256) == 6


def test_counts_go_with_the_newest_tokens_only(abi):
    lib, err, rows = abi.load(), C.create_string_buffer(256), _rows(abi)
    assert lib.fmha_kv4_read(_cache(abi), rows, rows, 3, 0, FAKE, None, err, 256) == 6 and "counts" in err.value.decode()


@pytest.mark.parametrize("change,message", [({"H": 3}, "1 to 16 times"), ({"H": 0}, "1 to 16 times"), ({"H": 34}, "1 to 16 times"), ({"out": None}, "out"), ({"out": FAKE + 4}, "out"),
                                            ({"weights": FAKE, "weights_width": 255}, "256 tokens"), ({"weights_in": FAKE}, "without weights"), ({"scale": 0.0}, "scale"),
                                            ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"S": 1 << 28, "H": 32}, "2^30"), ({"workspace": None}, "workspace"),
                                            ({"workspace": FAKE + 8}, "workspace"), ({"workspace_bytes": 100}, "workspace")])
def test_bad_attention_calls_are_refused(abi, change, message):
    lib, err = abi.load(), C.create_string_buffer(256)
    a = abi.Kv4AttendArgs(q=_rows(abi), out=FAKE, S=3, H=4, scale=1.0, workspace=FAKE, workspace_bytes=1 << 40)
    for k, v in change.items():
        setattr(a, k, v)
    assert lib.fmha_kv4_attend(_cache(abi), a, None, err, 256) == 6 and message in err.value.decode(), err.value
    assert lib.fmha_kv4_attend(_cache(abi), None, None, err, 256) == 6


@pytest.mark.parametrize("change,into,message", [({"keep": 0}, {}, "keep"), ({"keep": 257}, {}, "keep"), ({"keep": 10, "recent": 6, "first": 5}, {}, "exceed"), ({"weights": None}, {}, "weights"),
                                                 ({"kept": None}, {}, "kept"), ({"weights_width": 100}, {}, "cover"), ({"weights_out": FAKE, "weights_out_width": 9}, {}, "weights_out"),
                                                 ({}, {"B": 3}, "sequences, heads"), ({}, {"HK": 1}, "sequences, heads"), ({}, {"page": 32}, "sequences, heads"), ({}, {"table": FAKE}, "of its own"),
                                                 ({}, {"lengths": FAKE}, "of its own"), ({}, {"pool": None}, "must be given")])
def test_bad_evictions_are_refused(abi, change, into, message):
    lib, err = abi.load(), C.create_string_buffer(256)
    a = abi.Kv4EvictArgs(weights=FAKE, kept=FAKE, weights_width=256, keep=10)
    for k, v in change.items():
        setattr(a, k, v)
    target = _cache(abi, **{"table": 2 * FAKE, "lengths": 3 * FAKE, **into})
    assert lib.fmha_kv4_evict(_cache(abi), target, a, None, err, 256) == 6 and message in err.value.decode(), err.value


def test_nothing_to_do_is_no_error(abi):
    """No rows: nothing is launched, on a machine without a GPU too."""
    lib, err, rows = abi.load(), C.create_string_buffer(256), _rows(abi)
    assert lib.fmha_kv4_append(_cache(abi), rows, rows, 0, None, None, err, 256) == 0
    assert lib.fmha_kv4_read(_cache(abi), rows, rows, 0, 1, None, None, err, 256) == 0
    assert lib.fmha_kv4_attend(_cache(abi), abi.Kv4AttendArgs(q=rows, out=FAKE, S=0, H=2, scale=1.0), None, err, 256) == 0


def test_the_python_entry_wants_cuda_tensors():
    from amdgpu_rustdsl_b200 import Kv4Cache, kv4_pool
    pool = kv4_pool(4, 2, 64, device="cpu")
    assert tuple(pool.shape) == (4, 2, 64 * 136)
    with pytest.raises(ValueError, match="CUDA"):
        Kv4Cache(pool, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="16, 32, 64 or 128"):
        kv4_pool(4, 2, 48, device="cpu")
    with pytest.raises(ValueError, match="pool"):
        Kv4Cache(pool.view(torch.int8), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_the_reference_rounds_and_decodes_consistently():
    """The 64-bit restatement against itself: codes and scales decode to the values it rounds to, rounding is to nearest, and the nibble order is a permutation."""
    assert sorted(R.element_of_nibble().tolist()) == list(range(128))
    x = (torch.randn(64, 128, generator=torch.Generator().manual_seed(1)) * 3).bfloat16()
    codes, scales, value = R.encode(x)
    assert torch.equal(R.decode(codes, scales), value)
    step = R.power(scales.long() - 127).repeat_interleave(32, 1)
    grid = torch.tensor(R.GRID, dtype=torch.float64)
    nearest = ((x.double() / step).abs().clamp(max=6.0)[..., None] - grid).abs().amin(-1)
    assert torch.equal(((x.double().abs() / step).clamp(max=6.0) - (value.abs() / step)).abs(), nearest)
