"""Launches of attention over shared prefixes past 2^31 blocks are refused by what the kernel would really launch (asked of the library without a GPU)."""
import pytest

from test_shared_cpu import BASE, lib  # noqa: F401


@pytest.mark.parametrize("groups, splits, heads, kv, hd", [(30000, 120, 4000, 500, 128), (30000, 120, 4400, 1100, 128), (32767, 127, 8000, 1000, 64)])
def test_blocks_of_eight_rows_are_counted(lib, groups, splits, heads, kv, hd):  # noqa: F811
    code = lib.cima_attention_shared(BASE, 1, heads * hd, BASE, BASE, 8, 64, 2, BASE, BASE, BASE, BASE, BASE, groups, 2, BASE, BASE, splits, 1, BASE, heads * hd, 65535,
                                     heads, kv, hd, 0.125, 0.0, None, 0, None, 0, None)
    assert code < 0 and "blocks" in lib.cima_last_error().decode()
