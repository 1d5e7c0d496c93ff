"""The 8-bit cache's C ABI without a GPU: exports, and that wrong arguments are refused with a message before anything is launched or read."""
import ctypes as C
import os
import re

import pytest
import torch

from tests import kv8_reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 1 << 20   # an aligned address that nothing follows: every call here is refused


def test_every_declared_symbol_is_exported(abi):
    for header, names in (("kv8", abi.KV8_EXPORTS), ("rope", abi.ROPE_EXPORTS), ("pages", abi.PAGES_EXPORTS)):
        declared = set(re.findall(rf"\b(fmha_{header}_[a-z0-9_]+)\s*\(", open(os.path.join(ROOT, "include", f"fmha_{header}_abi.h")).read()))
        assert declared == set(names)
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
              ({"B": 1 << 16, "HK": 1 << 15}, "2^30"), ({"HK": 1 << 18}, "4 GiB")]


@pytest.mark.parametrize("change,message", BAD_CACHES)
def test_bad_caches_are_refused(abi, change, message):
    lib, err = abi.load(), C.create_string_buffer(256)
    rows = _rows(abi)
    assert lib.fmha_kv8_append(_cache(abi, **change), rows, rows, 3, None, None, err, 256) == 6 and message in err.value.decode()
    assert lib.fmha_kv8_read(_cache(abi, **change), rows, rows, 3, 0, None, None, err, 256) == 6 and message in err.value.decode()
    assert lib.fmha_kv8_attend(_cache(abi, **change), abi.Kv8AttendArgs(q=rows, out=FAKE, S=3, H=2, scale=1.0), None, err, 256) == 6 and message in err.value.decode()
    assert lib.fmha_kv8_attend_workspace(_cache(abi, **change), abi.Kv8AttendArgs(q=rows, out=FAKE, S=3, H=2, scale=1.0)) == 0


@pytest.mark.parametrize("change", [{"data": None}, {"data": FAKE + 2}, {"stride_b": 4}, {"stride_s": 129}, {"stride_h": 3}])
def test_bad_rows_are_refused(abi, change):
    lib, err = abi.load(), C.create_string_buffer(256)
    good, bad = _rows(abi), _rows(abi, **change)
    assert lib.fmha_kv8_append(_cache(abi), bad, good, 3, None, None, err, 256) == 6 and "k" in err.value.decode()
    assert lib.fmha_kv8_append(_cache(abi), good, bad, 3, None, None, err, 256) == 6 and "v" in err.value.decode()
    assert lib.fmha_kv8_read(_cache(abi), good, bad, 3, 1, None, None, err, 256) == 6
    assert lib.fmha_kv8_attend(_cache(abi), abi.Kv8AttendArgs(q=bad, out=FAKE, S=3, H=2, scale=1.0), None, err, 256) == 6


def test_too_many_rows_and_counts_without_last_are_refused(abi):
    lib, err, rows = abi.load(), C.create_string_buffer(256), _rows(abi)
    assert lib.fmha_kv8_append(_cache(abi), rows, rows, 1 << 29, None, None, err, 256) == 6 and "2^30" in err.value.decode()
    assert lib.fmha_kv8_read(_cache(abi), rows, rows, 1 << 29, 1, None, None, err, 256) == 6 and "2^30" in err.value.decode()
    assert lib.fmha_kv8_read(_cache(abi), rows, rows, 3, 0, FAKE, None, err, 256) == 6 and "counts" in err.value.decode()


@pytest.mark.parametrize("change,message", [({"H": 3}, "1 to 16 times"), ({"H": 0}, "1 to 16 times"), ({"H": 34}, "1 to 16 times"), ({"out": None}, "out"), ({"out": FAKE + 4}, "out"),
                                            ({"scale": 0.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"S": 1 << 28, "H": 32}, "2^30"), ({"workspace": None}, "workspace"),
                                            ({"workspace": FAKE + 8}, "workspace"), ({"workspace_bytes": 100}, "workspace")])
def test_bad_attention_calls_are_refused(abi, change, message):
    lib, err = abi.load(), C.create_string_buffer(256)
    a = abi.Kv8AttendArgs(q=_rows(abi), out=FAKE, S=3, H=4, scale=1.0, workspace=FAKE, workspace_bytes=1 << 40)
    for k, v in change.items():
        setattr(a, k, v)
    assert lib.fmha_kv8_attend(_cache(abi), a, None, err, 256) == 6 and message in err.value.decode(), err.value
    assert lib.fmha_kv8_attend(_cache(abi), None, None, err, 256) == 6


def test_out_may_be_q_only_packed(abi):
    lib, err = abi.load(), C.create_string_buffer(256)
    a = abi.Kv8AttendArgs(q=abi.Kv4Rows(FAKE, 6 * 4 * 128, 2 * 4 * 128, 128), out=FAKE, S=3, H=4, scale=1.0, workspace=FAKE, workspace_bytes=1 << 40)
    assert lib.fmha_kv8_attend(_cache(abi), a, None, err, 256) == 6 and "packed" in err.value.decode()


def test_nothing_to_do_is_no_error(abi):
    """No rows: nothing is launched, on a machine without a GPU too."""
    lib, err, rows = abi.load(), C.create_string_buffer(256), _rows(abi)
    assert lib.fmha_kv8_append(_cache(abi), rows, rows, 0, None, None, err, 256) == 0
    assert lib.fmha_kv8_read(_cache(abi), rows, rows, 0, 1, None, None, err, 256) == 0
    assert lib.fmha_kv8_attend(_cache(abi), abi.Kv8AttendArgs(q=rows, out=FAKE, S=0, H=2, scale=1.0), None, err, 256) == 0


def test_the_python_entry_wants_cuda_tensors():
    from amdgpu_rustdsl_b200 import Kv8Cache, kv8_pool
    pool = kv8_pool(4, 2, 64, device="cpu")
    assert tuple(pool.shape) == (4, 2, 64 * 257)
    with pytest.raises(ValueError, match="CUDA"):
        Kv8Cache(pool, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="16, 32, 64 or 128"):
        kv8_pool(4, 2, 48, device="cpu")
    with pytest.raises(ValueError, match="257"):
        Kv8Cache(pool.view(torch.int8), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_the_reference_rounds_and_places_as_it_says():
    """The 64-bit restatement against torch's e4m3 and against itself: every byte of a block's codes is one element's, K's and V's apart."""
    at = torch.cat([p.flatten() for p in R.PLACES])
    assert torch.equal(at.sort().values, torch.arange(4096)) and int(R.PLACES[0].max()) == 2047
    assert torch.equal(torch.arange(256).to(torch.uint8).view(torch.float8_e4m3fn).double().nan_to_num(7), R.grid().nan_to_num(7))
    y = torch.randn(1 << 16, dtype=torch.float64, generator=torch.Generator().manual_seed(1)) * torch.exp2(torch.linspace(-14, 8, 1 << 16, dtype=torch.float64))
    y = torch.cat([y, (R.grid()[:126] + R.grid()[1:127]) / 2]).clamp(-448, 448).float()   # and ties
    assert torch.equal(R.codes_of(y.double()), y.to(torch.float8_e4m3fn).view(torch.uint8))
    for largest in (0.0, 1e-40, 447.9, 448.0, 448.1, 7.0, 3e38):
        s = R.scale_of(largest)
        assert (largest <= 448 * s or s == 2.0 ** 119) and (s == 2.0 ** -90 or largest > 224 * s)
