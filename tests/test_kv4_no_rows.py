"""Calls of no rows: nothing to do, but for weights, which are the earlier ones."""
import ctypes as C

import pytest
import torch

from tests.test_kv4_host import FAKE, _cache


def test_rows_without_an_address(abi):
    """An empty tensor's address is 0."""
    lib, err = abi.load(), C.create_string_buffer(256)
    none = abi.Kv4Rows(None, 0, 256, 128)
    assert lib.fmha_kv4_append(_cache(abi), none, none, 0, None, None, err, 256) == 0
    assert lib.fmha_kv4_read(_cache(abi), none, none, 0, 1, None, None, err, 256) == 0
    a = abi.Kv4AttendArgs(q=none, out=None, S=0, H=2, scale=1.0)
    assert lib.fmha_kv4_attend(_cache(abi), a, None, err, 256) == 0
    a.weights = a.weights_in = FAKE
    assert lib.fmha_kv4_attend(_cache(abi), a, None, err, 256) == 0
    assert lib.fmha_kv4_append(_cache(abi), none, none, 1, None, None, err, 256) == 6 and "k" in err.value.decode()


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
def test_the_python_entries(causal):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4, kv4_append, kv4_read
    from tests.test_gpu_kv4 import make_cache
    cache = make_cache([300, 0, 47], 2, 32)
    before = cache.pool.clone()
    k = torch.empty(3, 0, 2, 128, dtype=torch.bfloat16, device="cuda")
    kv4_append(cache, k, k)
    kv4_read(cache, k, k)
    kv4_read(cache, k, k, last=True, counts=cache.lengths)
    q = torch.empty(3, 0, 8, 128, dtype=torch.bfloat16, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(3, 8, 0, device="cuda")
    fmha_fwd_kv4(q, cache, out, causal=causal, lse=lse)
    old, new, none = torch.rand(3, 2, cache.capacity, device="cuda"), torch.full((3, 2, cache.capacity), -7.0, device="cuda"), torch.full((3, 2, cache.capacity), -7.0, device="cuda")
    fmha_fwd_kv4(q, cache, out, causal=causal, lse=lse, weights=new, weights_in=old)
    fmha_fwd_kv4(q, cache, out, causal=causal, weights=none)
    live = (torch.arange(cache.capacity, device="cuda") < cache.lengths[:, None, None]).expand_as(old)
    assert torch.equal(new[live], old[live]) and (new[~live] == -7).all() and (none[live] == 0).all() and (none[~live] == -7).all()
    assert torch.equal(cache.pool, before)
