"""Numbers that do not fit the fields and registers they go into are refused, not cut."""
import ctypes as C
import types

import pytest
import torch

from tests.test_kv4_host import FAKE, _cache, _rows
from tests.test_workspaces_host import a_cache, no_gpu  # noqa: F401


def calls_nothing(*a):
    raise AssertionError("a call went out")


@pytest.fixture
def no_library(no_gpu, monkeypatch):  # noqa: F811
    from amdgpu_rustdsl_b200 import _abi
    lib = types.SimpleNamespace(fmha_kv4_evict=calls_nothing, fmha_kv4_append=calls_nothing, fmha_kv4_read=calls_nothing)
    monkeypatch.setattr(_abi, "load", lambda: lib)


@pytest.mark.parametrize("change", [dict(recent=1 << 32), dict(first=1 << 32), dict(keep=(1 << 32) + 16), dict(keep=65), dict(keep=1 << 31), dict(recent=(1 << 32) - 8, first=16), dict(recent=10, first=7)])
def test_evictions(no_library, change):
    from amdgpu_rustdsl_b200 import kv4
    with pytest.raises(ValueError, match="keep must be"):
        kv4.kv4_evict(a_cache(), torch.zeros(1, 1, 64), a_cache(), **{"keep": 16, **change})


def test_rows_of_a_stride_of_0(no_library):
    from amdgpu_rustdsl_b200 import kv4
    x = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16).expand(1, 1 << 32, 1, 128)
    for call in (kv4.kv4_append, kv4.kv4_read):
        with pytest.raises(ValueError, match="more than 2"):
            call(a_cache(), x, x)


def test_pages_of_4_gib(abi):
    """Pages of 128 tokens with the most heads that 32 bits hold pass this check (and stop at the next), those with one more do not."""
    lib, err, rows = abi.load(), C.create_string_buffer(256), _rows(abi)
    most = (2 ** 32 - 1) // (136 * 128)
    for heads, message in ((most + 1, "4 GiB"), (1 << 29, "4 GiB"), (most, "must be given")):
        cache = _cache(abi, HK=heads, B=1, page=128)
        assert lib.fmha_kv4_append(cache, abi.Kv4Rows(None, 8, 8, 8), rows, 3, None, None, err, 256) == 6 and message in err.value.decode()
        if heads > most:
            assert lib.fmha_kv4_attend(cache, abi.Kv4AttendArgs(q=rows, out=FAKE, S=3, H=heads, scale=1.0), None, err, 256) == 6 and message in err.value.decode()
            assert lib.fmha_kv4_evict(cache, cache, abi.Kv4EvictArgs(), None, err, 256) == 6 and message in err.value.decode()


@pytest.mark.parametrize("scale", [2.4e38, 3.3e38])
def test_scales_that_overflow_in_base_2(abi, scale):
    lib, err = abi.load(), C.create_string_buffer(256)
    a = abi.Kv4AttendArgs(q=_rows(abi), out=8 * FAKE, S=3, H=4, scale=scale, workspace=FAKE, workspace_bytes=1)
    assert lib.fmha_kv4_attend(_cache(abi), a, None, err, 256) == 6 and "scale must be" in err.value.decode()
    a.scale = 2.2e38
    assert lib.fmha_kv4_attend(_cache(abi), a, None, err, 256) == 6 and "workspace" in err.value.decode()
