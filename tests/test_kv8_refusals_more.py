"""CPU checks: more of what the 8-bit cache's entry points refuse before they look
for a device (device addresses here are never read)."""
import pytest

from test_kv8_refusals import ARG, K, S, T, V, X, Y, cache, rows

PAGED = dict(block_table=T, max_blocks=8, max_rows=8)      # 256 bytes of table


def test_rows_are_not_read_over_the_block_table():
    for n in ("k", "v"):
        for at in (T, T + 240, T - 1024, T - 5 * 1024 + 16):
            assert rows("read", cache(**PAGED), rows=(0, 1), **{n: at}) == ARG


@pytest.mark.parametrize("f", ["append", "read"])
def test_table_lies_apart_from_the_cache(f):
    for at in (K, V + 1024, S, S + 64 * 2 * 8 - 4, K - 252):
        assert rows(f, cache(**dict(PAGED, block_table=at)), rows=(0, 1), k=X, v=Y) == ARG
