"""What the operators for several answers to one prompt refuse, asked of the library itself without a GPU: a refusal comes before any CUDA call."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from cima_b200.csrc.build import library_path
    lib = ctypes.CDLL(library_path(build=True, verbose=False))
    lib.cima_last_error.restype = ctypes.c_char_p
    from cima_b200.kernels import _SIGNATURES
    for name in ("cima_copy_pages", "cima_attention_shared", "cima_attention_shared_tc", "cima_token_logprobs"):
        getattr(lib, name).argtypes = _SIGNATURES[name]
        getattr(lib, name).restype = ctypes.c_int
    return lib


BASE = 1 << 20          # an address that nothing reads


@pytest.mark.parametrize("plan, word", [
    ([(0, 4, 1)], "outside"), ([(4, 0, 1)], "outside"), ([(-1, 1, 1)], "outside"), ([(0, -1, 1)], "outside"), ([(0, 1, 17)], "positions"), ([(0, 1, -1)], "positions"),
    ([(0, 1, 1), (2, 1, 1)], "entry 1"), ([(0, 1, 1), (1, 2, 1)], "entry 1"), ([(1, 2, 1), (0, 1, 1)], "entry 1"), ([(3, 3, 1)], "reads"),
    ([(0, 1, 1)] + [(0, 2, 1), (0, 2, 1)], "entry 2"),
])
def test_bad_plans_of_copies(lib, plan, word):
    flat = (ctypes.c_int * (3 * len(plan)))(*[v for row in plan for v in row])
    assert lib.cima_copy_pages(BASE, 2, 4, 2, 16, 64, ctypes.addressof(flat), len(plan), None) < 0
    assert word in lib.cima_last_error().decode()


@pytest.mark.parametrize("args, word", [
    (dict(layers=0), "storage"), (dict(pages=0), "storage"), (dict(row=0), "storage"),
    (dict(row=1 << 28), "2\\^30"), (dict(row=1 << 62), "2\\^30"), (dict(layers=70000), "storage"),
])
def test_bad_storages_of_copies(lib, args, word):
    a = dict(base=BASE, layers=2, pages=4, segments=2, page=16, row=64) | args
    flat = (ctypes.c_int * 3)(0, 1, 1)
    code = lib.cima_copy_pages(a["base"], a["layers"], a["pages"], a["segments"], a["page"], a["row"], ctypes.addressof(flat), 1, None)
    assert code < 0
    import re
    assert re.search(word, lib.cima_last_error().decode())


def test_empty_calls_do_nothing(lib):
    assert lib.cima_copy_pages(None, 0, 0, 0, 0, 0, None, 0, None) == 0
    assert lib.cima_token_logprobs(None, 0, 5, None, None, None) == 0
    assert lib.cima_token_logprobs(BASE, 1, 0, BASE, BASE, None) < 0


@pytest.mark.parametrize("args, word", [
    (dict(planes=3), "planes"), (dict(page=32), "page size"), (dict(nh=5), "multiple"), (dict(groups=3), "groups"), (dict(most=3), "groups"), (dict(ps=0), "splits"),
    (dict(ps=100, os=29), "splits"), (dict(scratch=None), "scratch"), (dict(gate=300), "gate"), (dict(cache=BASE + 8), "aligned"), (dict(hd=72), "head_dim"),
    (dict(hd=144), "head_dim"), (dict(hd=132, dtype=0), "head_dim"), (dict(hd=66, dtype=0), "head_dim"), (dict(dtype=7), "dtype"), (dict(ld=257), "4-byte"),
])
def test_bad_arguments_of_shared_attention(lib, args, word):
    a = dict(dtype=1, ld=512, cache=BASE, page=64, planes=2, groups=1, most=2, scratch=BASE, ps=2, os=2, nh=4, nkv=2, hd=64, gate=0) | args
    code = lib.cima_attention_shared(BASE, a["dtype"], a["ld"], a["cache"], BASE, 8, a["page"], a["planes"], BASE, BASE, BASE, BASE, BASE, a["groups"], a["most"],
                                     a["scratch"], BASE, a["ps"], a["os"], BASE, 256, 2, a["nh"], a["nkv"], a["hd"], 0.125, 0.0, None, a["gate"], None, 0, None)
    assert code < 0
    assert word in lib.cima_last_error().decode()


@pytest.mark.parametrize("args, word", [
    (dict(planes=3), "planes"), (dict(page=32), "page size"), (dict(nh=5), "multiple"), (dict(groups=3), "groups"), (dict(ps=0), "splits"), (dict(scratch=None), "scratch"),
    (dict(gate=300), "gate"), (dict(cache=BASE + 8), "aligned"), (dict(hd=96), "head_dim"), (dict(ld=516), "aligned"), (dict(pages=0), "pages"),
    (dict(pages=1 << 24), "pages"), (dict(flag=None), "error flag"), (dict(scale=-0.125), "negative"), (dict(scale=float("nan")), "negative"),
])
def test_bad_arguments_of_shared_attention_on_tcgen05(lib, args, word):
    a = dict(ld=512, cache=BASE, pages=9, page=64, planes=2, groups=1, most=2, scratch=BASE, ps=2, os=2, nh=4, nkv=2, hd=64, gate=0, flag=BASE, scale=0.125) | args
    code = lib.cima_attention_shared_tc(BASE, a["ld"], a["cache"], a["pages"], BASE, 8, a["page"], a["planes"], BASE, BASE, BASE, BASE, BASE, a["groups"], a["most"],
                                        a["scratch"], BASE, a["ps"], a["os"], BASE, 256, 2, a["nh"], a["nkv"], a["hd"], a["scale"], 0.0, None, a["gate"], None, 0,
                                        a["flag"], None)
    assert code < 0
    assert word in lib.cima_last_error().decode()
