"""Caches of 4 and of 8 bits have the same fields: each call takes its own kind and refuses the other's, before it looks at anything."""
import pytest


def test_a_cache_of_the_other_kind_is_refused():
    import amdgpu_rustdsl_b200 as A
    four, eight = A.Kv4Cache.__new__(A.Kv4Cache), A.Kv8Cache.__new__(A.Kv8Cache)
    for call, kind in ((lambda: A.kv4_append(eight, None, None), "Kv4Cache, not Kv8Cache"), (lambda: A.kv4_read(eight, None, None), "Kv4Cache, not Kv8Cache"),
                       (lambda: A.fmha_fwd_kv4(None, eight, None), "Kv4Cache, not Kv8Cache"), (lambda: A.kv4_evict(eight, None, four, keep=1), "cache must be a Kv4Cache"),
                       (lambda: A.kv4_evict(four, None, eight, keep=1), "into must be a Kv4Cache"), (lambda: A.kv8_append(four, None, None), "Kv8Cache, not Kv4Cache"),
                       (lambda: A.kv8_read(four, None, None), "Kv8Cache, not Kv4Cache"), (lambda: A.fmha_fwd_kv8(None, four, None), "Kv8Cache, not Kv4Cache"),
                       (lambda: A.kv4_append(None, None, None), "not NoneType")):
        with pytest.raises(ValueError, match=kind):
            call()
