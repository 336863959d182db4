"""CPU checks: more of what the 8-bit cache's entry points refuse before they look
for a device (device addresses here are never read)."""
import ctypes as C

import pytest

import apus_hip as H
from test_kv8_refusals import ARG, K, S, T, UNS, V, X, Y, cache, rows

HIP = 4
PAGED = dict(block_table=T, max_blocks=8, max_rows=8)      # 256 bytes of table


def test_rows_are_not_read_over_the_block_table():
    for n in ("k", "v"):
        for at in (T, T + 240, T - 1024, T - 5 * 1024 + 16):
            assert rows("read", cache(**PAGED), rows=(0, 1), **{n: at}) == ARG


@pytest.mark.parametrize("f", ["append", "read"])
def test_table_lies_apart_from_the_cache(f):
    for at in (K, V + 1024, S, S + 64 * 2 * 8 - 4, K - 252):
        assert rows(f, cache(**dict(PAGED, block_table=at)), rows=(0, 1), k=X, v=Y) == ARG


@pytest.mark.parametrize("f", ["append", "read"])
@pytest.mark.parametrize("nkv,lens", [(2, (1 << 26,)), (1, (1 << 27,)), (1024, (32 * 2048, 32 * 2048)), (1, (1 << 26, 1 << 26))])
def test_no_more_blocks_than_a_launch_has(f, nkv, lens):
    """2^22 (block, head) pairs and more: refused, not left to fail at the launch."""
    cu = (0,) + tuple(sum(lens[:i + 1]) for i in range(len(lens)))
    far = 1 << 46                          # (arrays of terabytes, apart)
    c = cache(k=far, v=2 * far, scale=3 * far, blocks=1 << 23, max_blocks=1 << 22, max_rows=2)
    assert rows(f, c, nkv=nkv, B=len(lens), cu=cu, pos=(0,) * len(lens), k=4 * far, ldk=nkv * 256, v=6 * far,
                ldv=nkv * 256) == UNS


def pool(name, nlayers=1, nkv=2, d=256, nblocks=4, max_rows=2, max_blocks=2):
    out = C.c_void_p(1)
    rc = getattr(H.load(), f"apus_hip_{name}_pool_create")(*map(C.c_size_t, (nlayers, nkv, d, nblocks, max_rows, max_blocks)),
                                                           C.byref(out))
    assert rc == 0 or not out.value
    return rc


def test_pool_sizes_that_its_calls_refuse():
    assert pool("kv8", nkv=1025) == UNS and pool("kv8", max_blocks=(1 << 25) + 1) == UNS
    for name in ("kv", "kv8"):
        assert pool(name, nkv=1 << 50) == UNS              # (bytes of a block past 64 bits)
        for kw in (dict(nlayers=0), dict(nkv=0), dict(d=128), dict(nblocks=0), dict(max_rows=1 << 31), dict(max_blocks=0)):
            assert pool(name, **kw) == ARG


@pytest.mark.parametrize("name", ["kv", "kv8"])
def test_pool_past_the_hosts_memory(name):
    """Bookkeeping that no host can hold is an error, not an exception."""
    most = (1 << 31) - 1
    assert pool(name, max_rows=most, max_blocks=1 << 25) == HIP
    assert pool(name, nlayers=1 << 60) == HIP
