"""The scratch of an attention over shared prefixes is the call's own until its kernels are launched (no GPU: the library's entries are stand-ins that look)."""
import weakref
from types import SimpleNamespace

import pytest
import torch

from shared_cases import PAGE, shared_case
from cima_b200 import kernels
from cima_b200.cache import LayerKV, SharedPrefixes
from cima_b200.kernels import Kernels


class Watched:
    """Every tensor that torch.empty, torch.zeros and new_empty made, for as long as it lives."""

    def __init__(self, monkeypatch):
        self.made = []
        for owner, name in ((torch, "empty"), (torch, "zeros"), (torch.Tensor, "new_empty"), (torch.Tensor, "new_zeros")):
            monkeypatch.setattr(owner, name, self.wrapped(getattr(owner, name)))

    def wrapped(self, make):
        def made(*args, **kw):
            t = make(*args, **kw)
            self.made.append((weakref.ref(t), t.data_ptr(), t.numel() * t.element_size()))
            return t
        return made

    def owner(self, address):
        return [i for i, (t, at, n) in enumerate(self.made) if t() is not None and at <= address < at + n]


@pytest.mark.parametrize("dtype, tc", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.bfloat16, None), (torch.float32, None)])
def test_scratch_lives_until_the_launch(monkeypatch, dtype, tc):
    c = shared_case([5], [3], [1, 64, 70], 28, 4, 64, dtype, alone=[9], device="cpu")
    K, seen = object.__new__(Kernels), []
    K.profile = K._error_flag = None                                     # a fresh one: the flag is made by this call where it needs one
    K.launches = 0
    monkeypatch.setattr(kernels, "_current_device", lambda: -1)
    monkeypatch.setattr(kernels, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(Kernels, "_need", staticmethod(lambda *a: None))
    watched = Watched(monkeypatch)

    def entry(name):
        def call(*args):
            part_o, part_ml = args[15:17]
            flag = args[-2] if name.endswith("_tc") else None
            seen.append(name)
            assert watched.owner(part_o) and watched.owner(part_o) == watched.owner(part_ml), "the scratch was given back before the launch"
            if flag is not None:
                assert watched.owner(flag) and watched.owner(flag) != watched.owner(part_o)
            return 0
        return call

    K.lib = SimpleNamespace(cima_attention_shared=entry("cima_attention_shared"), cima_attention_shared_tc=entry("cima_attention_shared_tc"))
    out = torch.empty(c.B, c.heads * c.hd, dtype=dtype)
    K.attention_shared(c.qkv, LayerKV(c.storage, c.table, PAGE, 0, 0, 0), c.slot, c.len, SharedPrefixes(c.order, c.own_page, c.groups, c.most), out, c.heads,
                       c.kv_heads, c.hd, c.scale, c.max_len, tc=tc)
    assert seen == ["cima_attention_shared_tc" if tc is not False and dtype is torch.bfloat16 else "cima_attention_shared"]
