"""Arguments of the 4-bit cache's operators that share memory where a kernel could read what another of its threads has written: refused on the host, before anything is launched."""
import ctypes as C

import pytest

from tests.test_kv4_host import FAKE, _cache, _rows

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


def attend(abi, S=3, H=4, **change):
    lib, err = abi.load(), C.create_string_buffer(256)
    q = abi.Kv4Rows(FAKE, S * H * 128, H * 128, 128)
    a = abi.Kv4AttendArgs(q=q, out=64 * FAKE, S=S, H=H, scale=1.0, workspace=32 * FAKE, workspace_bytes=1 << 40, weights=2 * FAKE, weights_in=4 * FAKE, weights_width=WIDTH)
    for k, v in change.items():
        setattr(a, k, v)
    return lib.fmha_kv4_attend(_cache(abi), a, None, err, 256), err.value.decode()


@pytest.mark.parametrize("offset", [4, -4, 4 * B * HK * WIDTH - 4, 4 - 4 * B * HK * WIDTH])
def test_weights_that_lie_askew_over_the_earlier_ones(abi, offset):
    rc, message = attend(abi, weights_in=2 * FAKE + offset)
    assert rc == 6 and "share no memory" in message


def test_attention_in_the_place_of_strided_queries(abi):
    for stride in ("stride_b", "stride_s", "stride_h"):
        q = _rows(abi, stride_b=3 * 4 * 128, stride_s=4 * 128, stride_h=128)
        setattr(q, stride, getattr(q, stride) + 128)
        rc, message = attend(abi, q=q, out=FAKE, weights=None, weights_in=None)
        assert rc == 6 and "only where q is packed" in message


def test_attention_in_the_place_of_queries_that_the_weights_go_by(abi):
    rc, message = attend(abi, S=5, out=FAKE)   # 10 rows of a KV head
    assert rc == 6 and "more than 8 rows" in message
