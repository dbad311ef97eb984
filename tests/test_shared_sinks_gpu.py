"""Attention over shared prefixes: sinks and scores over the range of float32's exponent and beyond, against 64 bits."""
import pytest
import torch

from shared_cases import PAGE, shared_case, shared_reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from cima_b200.kernels import Kernels
    return Kernels(verbose=False)


ROADS = [("tc", [26, 3], 14, 2, 64, torch.bfloat16), ("tc128", [40], 12, 2, 128, torch.bfloat16), ("near", [2], 14, 2, 64, torch.bfloat16),
         ("mma", [9], 8, 2, 96, torch.bfloat16), ("f32", [6], 14, 2, 64, torch.float32)]


@pytest.mark.parametrize("scores", [-120.0, 0.0, 120.0])
@pytest.mark.parametrize("sink", [-120.0, -90.0, 0.0, 90.0, 120.0])
@pytest.mark.parametrize("road", ROADS, ids=[r[0] for r in ROADS])
def test_stored_sinks_beside_scores_far_from_zero(K, road, sink, scores):
    """Each head's sink near ``sink``, its scores near ``scores`` (the first value of every query and key is set so), and the other way round."""
    from cima_b200.cache import LayerKV, SharedPrefixes
    _, counts, heads, kv, hd, dtype = road
    c = shared_case(counts, [5] * len(counts), [1, 64, 90], heads, kv, hd, dtype, alone=[70], seed=hd)
    c.qkv[:, :heads * hd:hd] = scores / 32.0
    c.storage[:, 0, ..., 0] = 32.0 / c.scale
    c.sink = c.sink + sink
    L = LayerKV(c.storage, c.table, PAGE, 0, 0, 0, c.planes)
    plan = SharedPrefixes(c.order, c.own_page, c.groups, c.most)
    for more in (dict(head_sink=c.sink), dict(sink=3.0), dict()):
        want, tol = shared_reference(c, **more)
        out = torch.empty(c.B, heads * hd, dtype=dtype, device="cuda")
        K.attention_shared(c.qkv, L, c.slot, c.len, plan, out, heads, kv, hd, c.scale, c.max_len, **more)
        off = (out.double().cpu() - want).abs()
        assert (off <= tol).all(), (more.keys(), float((off / tol).max()))


@pytest.mark.parametrize("road", ROADS, ids=[r[0] for r in ROADS])
def test_infinite_sinks(K, road):
    """A sink of -inf is none; one of +inf leaves the values no weight."""
    from cima_b200.cache import LayerKV, SharedPrefixes
    _, counts, heads, kv, hd, dtype = road
    c = shared_case(counts, [5] * len(counts), [1, 64, 90], heads, kv, hd, dtype, alone=[70], seed=hd)
    L, plan = LayerKV(c.storage, c.table, PAGE, 0, 0, 0, c.planes), SharedPrefixes(c.order, c.own_page, c.groups, c.most)

    def run(**more):
        out = torch.empty(c.B, heads * hd, dtype=dtype, device="cuda")
        K.attention_shared(c.qkv, L, c.slot, c.len, plan, out, heads, kv, hd, c.scale, c.max_len, **more)
        return out

    assert torch.equal(run(head_sink=torch.full((heads,), -float("inf"), device="cuda")), run())
    assert (run(head_sink=torch.full((heads,), float("inf"), device="cuda")) == 0).all()
    assert (run(head_sink=torch.full((heads,), 3e38, device="cuda")) == 0).all()
