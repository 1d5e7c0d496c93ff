"""Arguments of the 4-bit cache's operators that share memory where a kernel could read what another of its threads has written: refused on the host, before anything is launched."""
import ctypes as C

import pytest

from tests.test_kv4_host import FAKE, _cache

B, HK, WIDTH = 2, 2, 256   # of _cache: 4 pages of 64 tokens


def evict(abi, **change):
    lib, err = abi.load(), C.create_string_buffer(256)
    a = abi.Kv4EvictArgs(weights=FAKE, kept=16 * FAKE, weights_width=WIDTH, keep=10, weights_out_width=WIDTH)
    for k, v in change.items():
        setattr(a, k, v)
    return lib.fmha_kv4_evict(_cache(abi), _cache(abi, table=2 * FAKE, lengths=3 * FAKE), a, None, err, 256), err.value.decode()


@pytest.mark.parametrize("offset,width", [(0, WIDTH), (4, WIDTH), (-4, WIDTH), (4 * B * HK * WIDTH - 4, WIDTH), (4 - 4 * B * HK * WIDTH, WIDTH), (1024, 10), (4 - 4 * B * HK * 10, 10)])
def test_evictions_into_the_weights_they_go_by(abi, offset, width):
    rc, message = evict(abi, weights_out=FAKE + offset, weights_out_width=width)
    assert rc == 6 and "weights_out must not share memory" in message
