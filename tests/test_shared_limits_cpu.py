"""Launches of attention over shared prefixes past 2^31 blocks are refused by what the kernel would really launch (asked of the library without a GPU)."""
import pytest

from test_shared_cpu import BASE, lib  # noqa: F401


@pytest.mark.parametrize("groups, splits, heads, kv, hd", [(30000, 120, 4000, 500, 128), (30000, 120, 4400, 1100, 128), (32767, 127, 8000, 1000, 64)])
def test_blocks_of_eight_rows_are_counted(lib, groups, splits, heads, kv, hd):  # noqa: F811
    code = lib.cima_attention_shared(BASE, 1, heads * hd, BASE, BASE, 8, 64, 2, BASE, BASE, BASE, BASE, BASE, groups, 2, BASE, BASE, splits, 1, BASE, heads * hd, 65535,
                                     heads, kv, hd, 0.125, 0.0, None, 0, None, 0, None)
    assert code < 0 and "blocks" in lib.cima_last_error().decode()


def test_a_result_of_other_dimensions_is_refused_by_name(monkeypatch):
    import torch
    from shared_cases import PAGE, shared_case
    from cima_b200 import kernels
    from cima_b200.cache import LayerKV, SharedPrefixes
    c = shared_case([2], [1], [1], 4, 2, 64, torch.bfloat16, device="cpu")
    monkeypatch.setattr(kernels, "_current_device", lambda: -1)
    K = object.__new__(kernels.Kernels)
    for out in (torch.empty(c.B * 256, dtype=torch.bfloat16), torch.empty(c.B, 4, 64, dtype=torch.bfloat16)):
        with pytest.raises(kernels.KernelError):
            K.attention_shared(c.qkv, LayerKV(c.storage, c.table, PAGE, 0, 0, 0), c.slot, c.len, SharedPrefixes(c.order, c.own_page, c.groups, c.most), out, 4, 2, 64, 0.125)
