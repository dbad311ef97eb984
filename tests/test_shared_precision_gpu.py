"""Attention over shared prefixes is no further from 64 bits than the one-token attention that it stands for."""
import pytest
import torch

from shared_cases import PAGE, shared_case, shared_reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from cima_b200.kernels import Kernels
    return Kernels(verbose=False)


def relative(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


def both(K, c, **more):
    """Relative errors against float64 of (the shared kernel, the split kernel at 64 splits, whose sums are the shortest)."""
    from cima_b200.cache import LayerKV, SharedPrefixes
    kv = LayerKV(c.storage, c.table, PAGE, 0, 0, 0, c.planes)
    want, _ = shared_reference(c)
    out = torch.empty(c.B, c.heads * c.hd, dtype=c.dtype, device="cuda")
    K.attention_shared(c.qkv, kv, c.slot, c.len, SharedPrefixes(c.order, c.own_page, c.groups, c.most), out, c.heads, c.kv_heads, c.hd, c.scale, c.max_len, **more)
    shared = relative(out, want)
    K.attention_decode(c.qkv, kv, c.slot, c.len, out, c.heads, c.kv_heads, c.hd, c.scale, 0, c.max_len, n_splits=64)
    return shared, relative(out, want)


@pytest.mark.parametrize("spread", [1.0, 3.0])
@pytest.mark.parametrize("signs", ["mixed", "one"])
@pytest.mark.parametrize("counts, prefix, own, heads, kv, hd, more", [
    ([8], [32], [1, 64, 65, 100], 28, 4, 128, {}),
    ([48], [40], [1, 130], 28, 4, 128, {}),
    ([48], [40], [1, 130], 28, 4, 128, dict(splits=(1, 1))),
    ([6, 6], [63, 20], [17], 12, 2, 128, {}),
    ([33], [30], [5, 64], 14, 2, 64, {}),
    ([40], [30], [5, 64], 14, 2, 64, dict(splits=(1, 1))),
    ([2], [30], [5, 64], 14, 2, 64, {}),
    ([2], [30], [5, 64], 28, 4, 128, {}),
    ([24], [40], [5, 64], 8, 2, 96, {}),
    ([4], [40], [5, 64], 8, 2, 48, {}),
])
def test_as_near_to_64_bits_as_the_splits(K, counts, prefix, own, heads, kv, hd, more, signs, spread):
    """Flat rows and rows of few large probabilities, values of mixed and of one sign (2 % for what the rounding of the result leaves to chance)."""
    c = shared_case(counts, prefix, own, heads, kv, hd, torch.bfloat16, seed=hd)
    c.storage[~(c.storage.abs() < 100)] = 0.0            # (what lies behind a sequence's end: the split kernel multiplies it by 0)
    if signs == "one":
        c.storage[:, 1] = c.storage[:, 1].abs()
    c.qkv[:, :heads * hd] *= spread
    shared, splits = both(K, c, **more)
    assert K.device_errors() == 0
    print(f"{shared:.3e} {splits:.3e}")
    assert shared <= 1.02 * splits, (shared, splits)
