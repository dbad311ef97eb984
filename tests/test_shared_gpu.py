"""Attention over shared prefixes, copies of pages and log-probabilities of tokens against plain implementations in 64 bits."""
import math

import pytest
import torch

from shared_cases import PAGE, logprob_reference, shared_case, shared_reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from cima_b200.kernels import Kernels
    return Kernels(verbose=False)


def run_shared(K, c, splits=None, **more):
    from cima_b200.cache import LayerKV, SharedPrefixes
    kv = LayerKV(c.storage, c.table, PAGE, 0, 0, 0, c.planes)
    out = torch.full((c.B, c.heads * c.hd), 7.0, dtype=c.dtype, device=c.qkv.device)
    K.attention_shared(c.qkv, kv, c.slot, c.len, SharedPrefixes(c.order, c.own_page, c.groups, c.most), out, c.heads, c.kv_heads, c.hd, c.scale,
                       c.max_len, splits=splits, **more)
    return out


def check(got, want, tol):
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got.float()).all()
    assert (off <= tol).all(), f"{int((off > tol).sum())} values, worst {float((off / tol).max()):.3g} times the bound"


SIZES = [
    # counts, prefix pages, own positions, alone, heads, kv, hd
    ([2], [1], [1], [], 1, 1, 64),
    ([2], [5], [1, 40], [], 14, 2, 64),
    ([8], [32], [1, 63, 64, 65, 100], [], 28, 4, 128),
    ([3], [3], [17], [1, 64, 700], 4, 2, 16),
    ([2, 5, 9], [1, 4, 2], [1, 2, 130, 64], [5], 12, 2, 128),
    ([19], [3], [33, 1], [], 40, 8, 128),
    ([70], [9], [1, 200, 64], [], 28, 4, 128),
    ([33], [7], [5, 64], [900], 40, 2, 64),
    ([2, 2], [2, 6], [300, 9], [], 6, 3, 48),
    ([4], [2], [77], [3], 8, 2, 112),
    ([4], [2], [77], [3], 5, 1, 96),
    ([], [], [], [1, 65, 128], 8, 2, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("planes", [2, 1])
@pytest.mark.parametrize("size", SIZES, ids=[str(i) for i in range(len(SIZES))])
def test_shared_attention(K, size, planes, dtype):
    counts, prefix, own, alone, heads, kv, hd = size
    c = shared_case(counts, prefix, own, heads, kv, hd, dtype, planes=planes, alone=alone, seed=len(counts) + heads)
    check(run_shared(K, c), *shared_reference(c))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("what", ["sink", "head_sink", "slopes", "gate", "all"])
@pytest.mark.parametrize("hd", [64, 128])
def test_shared_attention_forms(K, what, dtype, hd):
    c = shared_case([6, 2], [3, 1], [1, 64, 90], 14, 2, hd, dtype, alone=[70], gate=what in ("gate", "all"), seed=11)
    more = {}
    if what == "sink":
        more["sink"] = 2.0
    if what in ("head_sink", "all"):
        more["head_sink"] = c.sink
    if what in ("slopes", "all"):
        more["slopes"] = c.slopes
    if what in ("gate", "all"):
        more["gate_col"] = c.gate_col
    check(run_shared(K, c, **more), *shared_reference(c, **more))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("splits", [(1, 1), (3, 2), (64, 32), (64, 64), (1, 127)])
def test_shared_attention_splits(K, splits, dtype):
    c = shared_case([5], [11], [1, 64, 150], 12, 2, 64, dtype, alone=[1, 500], seed=3)
    check(run_shared(K, c, splits=splits), *shared_reference(c))


TC_SIZES = [([2], [1], [1], [], 1, 1, 64), ([8], [32], [1, 63, 64, 65, 100], [], 28, 4, 128), ([2, 5, 19], [1, 4, 2], [1, 2, 130, 64], [5], 12, 2, 128),
            ([70], [9], [1, 200, 64], [], 28, 4, 128), ([33], [7], [5, 64], [900], 40, 2, 64), ([128], [3], [1], [], 8, 8, 64), ([129], [2], [7], [], 8, 8, 128)]


@pytest.mark.parametrize("planes", [2, 1])
@pytest.mark.parametrize("size", TC_SIZES, ids=[str(i) for i in range(len(TC_SIZES))])
@pytest.mark.parametrize("splits", [None, (1, 1), (7, 3)])
def test_shared_attention_on_tcgen05(K, size, planes, splits):
    counts, prefix, own, alone, heads, kv, hd = size
    c = shared_case(counts, prefix, own, heads, kv, hd, torch.bfloat16, planes=planes, alone=alone, seed=len(counts) + heads)
    check(run_shared(K, c, splits=splits, tc=True), *shared_reference(c))
    assert K.device_errors() == 0


def test_many_launches_on_tcgen05_in_a_row(K):
    """Some thousand launches as a recorded step makes them, each let begin while the kernel before it ends: no bounded wait runs out (one in
    some thousand did, where a warp asked for a phase that two later ones had overtaken), and every result is the first one's."""
    c = shared_case([48], [32], [100, 1, 64, 130], 28, 4, 128, torch.bfloat16, seed=2)
    want = run_shared(K, c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = [run_shared(K, c, early=True) for _ in range(40)]
    K.device_errors()
    for _ in range(100):
        g.replay()
    torch.cuda.synchronize()
    assert K.device_errors() == 0
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("hd", [64, 128])
def test_shared_attention_forms_on_tcgen05(K, hd):
    c = shared_case([26, 2], [3, 1], [1, 64, 90], 14, 2, hd, torch.bfloat16, alone=[70], gate=True, seed=11)
    more = dict(head_sink=c.sink, slopes=c.slopes, gate_col=c.gate_col)
    check(run_shared(K, c, tc=True, **more), *shared_reference(c, **more))
    check(run_shared(K, c, tc=True, sink=3.0), *shared_reference(c, sink=3.0))
    c.storage[:, 0] *= 20.0                               # scores of some hundred: the reference point moves often
    check(run_shared(K, c, tc=True), *shared_reference(c))


def test_shared_attention_large_scores(K):
    """Scores of several hundred, of both signs: the parts' maxima lie far from one another and a part's weight may vanish."""
    c = shared_case([4], [4], [70, 3], 8, 2, 64, torch.float32, seed=9)
    c.storage[:, 0] *= 30.0
    check(run_shared(K, c), *shared_reference(c))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("hd", [48, 64, 96, 128])
@pytest.mark.parametrize("splits", [None, (1, 1), (2, 2), (3, 4), (2, 120)])
def test_shared_attention_begun_early(K, splits, hd, dtype):
    """A launch that reads its pages ahead of the kernel before it, which may still write each sequence's newest position: at the end of a page, at
    its beginning, alone in the sequence; in the last of its own pages' splits or the only one."""
    for counts in ([3], [40]):
        c = shared_case(counts, [5], [1, 64, 65, 128, 300, 640], 8, 2, hd, dtype, alone=[1, 64, 65, 500], gate=True, seed=hd)
        check(run_shared(K, c, splits=splits, early=True, gate_col=c.gate_col, slopes=c.slopes), *shared_reference(c, gate_col=c.gate_col, slopes=c.slopes))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_shared_attention_behind_the_write_of_its_newest_position(K, hd, dtype):
    """The kernel that turns and stores a step's new keys, then at once the attention that begins early, many times over: what it reads is new."""
    for counts, splits in ([3], None), ([40], None), ([40], (3, 4)):
        c = shared_case(counts, [5], [1, 64, 65, 200], 8, 2, hd, dtype, alone=[64, 130], seed=hd)
        first = run_shared(K, c, splits=splits)
        cols = slice(0, c.heads * hd)
        pages = c.table[c.slot.long(), (c.len.long() - 1) // PAGE].long()
        at = (c.len.long() - 1) % PAGE
        now = c.storage[pages, :, :, at].clone()
        wrong, q = torch.full_like(now, 50.0), c.qkv[:, cols].clone()
        g = torch.cuda.CUDAGraph()
        got = torch.empty_like(first)
        run = lambda: got.copy_(run_shared(K, c, splits=splits, early=True))     # noqa: E731
        run()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            c.storage[pages, :, :, at] = wrong
            c.qkv[:, cols] = 3.0
            c.storage[pages, :, :, at] = now
            c.qkv[:, cols] = q
            run()
        for _ in range(20):
            g.replay()
            assert torch.equal(got, first)
        check(got, *shared_reference(c))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("counts", [[3], [7], [40]])
def test_shared_attention_of_rows_at_odd_places(K, counts, hd):
    """Rows that begin 4 bytes behind a 16-byte boundary take the kernels that ask for no more."""
    c = shared_case(counts, [3], [1, 64, 90], 4, 1, hd, torch.bfloat16, alone=[70], seed=4)
    buf = torch.empty(c.qkv.numel() + 8, dtype=torch.bfloat16, device="cuda")
    moved = buf[2:2 + c.qkv.numel()].view_as(c.qkv)
    moved.copy_(c.qkv)
    c.qkv = moved
    check(run_shared(K, c), *shared_reference(c))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_shared_attention_of_a_negative_scale(K, dtype):
    c = shared_case([12], [4], [1, 64, 90], 14, 2, 64, dtype, alone=[70], seed=4)
    c.scale = -c.scale
    check(run_shared(K, c), *shared_reference(c))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("hd", [48, 64, 128])
@pytest.mark.parametrize("early", [False, True])
@pytest.mark.parametrize("counts", [[3], [40]])
def test_shared_attention_of_an_empty_sequence(K, counts, early, hd, dtype):
    """A sequence without a position gives zeros, and the others what they gave."""
    c = shared_case(counts, [5], [1, 64, 200], 8, 2, hd, dtype, alone=[64, 70, 1], gate=True, seed=hd)
    more = dict(early=early, gate_col=c.gate_col, slopes=c.slopes, splits=(3, 2))
    want = run_shared(K, c, **more)
    empty = int((c.own_page == 0).nonzero()[1])
    c.len[empty] = 0
    got = run_shared(K, c, **more)
    assert (got[empty] == 0).all()
    keep = torch.arange(c.B, device="cuda") != empty
    assert torch.equal(got[keep], want[keep])


def test_shared_attention_of_no_sequences(K):
    c = shared_case([3], [5], [1, 64], 8, 2, 64, torch.bfloat16)
    c.qkv, c.B = c.qkv[:0], 0
    assert run_shared(K, c).shape == (0, 512)


def test_padded_groups_and_their_order(K):
    """Groups without sequences (a recorded step's spare places) take no part; the result does not depend on which spare places there are."""
    c = shared_case([3, 4], [2, 3], [1, 65], 14, 2, 64, torch.bfloat16, seed=5)
    want = run_shared(K, c, splits=(4, 2))
    c.groups = torch.cat([c.groups, torch.zeros(3, 3, dtype=torch.int32, device="cuda")])
    assert torch.equal(run_shared(K, c, splits=(4, 2)), want)


def test_shared_equals_unshared(K):
    """The same batch without its groups (each sequence reads all its pages itself): within twice the bound of each other."""
    c = shared_case([6], [9], [1, 64, 90], 28, 4, 128, torch.bfloat16, alone=[30], seed=6)
    want, tol = shared_reference(c)
    a = run_shared(K, c)
    c.groups, c.own_page, c.most = c.groups[:0], torch.zeros_like(c.own_page), 0
    check(run_shared(K, c), a.double().cpu(), 2 * tol)


def test_shared_attention_replayed_and_on_a_stream(K):
    c = shared_case([7], [6], [1, 64, 90], 14, 2, 64, torch.bfloat16, seed=8)
    want = run_shared(K, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run_shared(K, c)
    side.synchronize()
    assert torch.equal(other, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run_shared(K, c)
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    # what a replay reads on the device may change: shorter sequences, other groups
    c2 = shared_case([7], [6], [2, 11, 65], 14, 2, 64, torch.bfloat16, seed=21)
    for n in ("qkv", "slot", "len", "order", "own_page", "groups"):
        getattr(c, n).copy_(getattr(c2, n))
    assert c.storage.shape[0] >= c2.storage.shape[0]
    c.storage[:c2.storage.shape[0]].copy_(c2.storage)
    c.table[:, :c2.table.shape[1]].copy_(c2.table)
    g.replay()
    check(out, *shared_reference(c2))


def test_shared_attention_refusals(K):
    from cima_b200.cache import LayerKV, SharedPrefixes
    from cima_b200.kernels import KernelError
    c = shared_case([2], [1], [1], 4, 2, 64, torch.bfloat16)
    plan = SharedPrefixes(c.order, c.own_page, c.groups, c.most)
    out = torch.empty(c.B, 256, dtype=torch.bfloat16, device="cuda")

    def call(kv=None, shared=plan, out=out, heads=4, slot=c.slot, splits=None, qkv=c.qkv, **more):
        K.attention_shared(qkv, kv or LayerKV(c.storage, c.table, PAGE, 0, 0, 0), slot, c.len, shared, out, heads, 2, 64, 0.125, splits=splits, **more)

    for kw, word in [(dict(out=out[:, :128].contiguous()), "do not fit"), (dict(kv=LayerKV(c.storage, c.table, PAGE, 3, 128, 0)), "window"),
                     (dict(slot=c.slot.long()), "expected"), (dict(slot=c.slot[:1]), "entries"), (dict(splits=(0, 1)), "splits"), (dict(splits=(64, 65)), "splits"),
                     (dict(shared=SharedPrefixes(c.order, c.own_page, c.groups, 5)), "groups"), (dict(gate_col=c.qkv.shape[1] - 8), "gate"),
                     (dict(shared=SharedPrefixes(c.order.cpu(), c.own_page, c.groups, 2)), "GPU tensors"), (dict(heads=3, out=out[:, :192].contiguous()), "multiple"),
                     (dict(heads=3, out=out[:, :192].contiguous(), tc=True), "multiple"), (dict(splits=(64, 65), tc=True), "splits"),
                     (dict(kv=LayerKV(c.storage.half(), c.table, PAGE, 0, 0, 0)), "expected"), (dict(slopes=c.slopes[:2]), "slopes"),
                     (dict(shared=SharedPrefixes(c.order, c.own_page, c.groups[:, :2].contiguous(), 2)), "groups")]:
        with pytest.raises(KernelError, match=word):
            call(**kw)
    call()


# ---------------------------------------------------------------------------------------------- pages
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.float16, torch.uint8])
@pytest.mark.parametrize("shape", [(1, 9, 1, 1, 64, 16), (3, 40, 2, 4, 64, 128), (24, 700, 2, 2, 64, 8), (1, 6, 1, 1, 1, 1), (2, 7, 1, 3, 16, 3), (1, 30, 1, 1, 1, 500)])
def test_copy_pages(K, shape, dtype):
    gen = torch.Generator().manual_seed(1)
    x = torch.randint(-1 << 14, 1 << 14, shape, generator=gen)
    x = x.to(dtype)
    n = (shape[1] - 1) // 2
    ids = torch.randperm(shape[1], generator=gen)
    fill = torch.randint(0, shape[4] + 1, (n,), generator=gen)
    fill[0] = shape[4]
    plan = torch.stack([ids[:n], ids[n:2 * n], fill], 1).int()
    plan[n // 2:, 0] = plan[0, 0]                         # one page for several others
    want = x.clone()
    for a, b, k in plan.tolist():
        want[:, b, :, :, :k] = x[:, a, :, :, :k]
    got = x.cuda()
    K.copy_pages(got, plan)
    assert torch.equal(got.cpu(), want)
    K.copy_pages(got, plan[:0])
    assert torch.equal(got.cpu(), want)


def test_copy_pages_of_a_large_storage(K):
    """Offsets beyond 2^32 bytes and 2^31 elements."""
    x = torch.zeros(2, 1200, 2, 8, PAGE, 1024, dtype=torch.int16, device="cuda")
    assert x.numel() > 2 ** 31
    x[1, 1199] = 5
    K.copy_pages(x, torch.tensor([[1199, 1198, 33], [1199, 0, 64]], dtype=torch.int32))
    assert (x[1, 1198, :, :, :33] == 5).all() and (x[1, 1198, :, :, 33:] == 0).all() and (x[1, 0] == 5).all() and (x[0] == 0).all() and (x[1, 1:1198] == 0).all()


def test_copy_pages_of_storage_at_odd_places(K):
    """Storage that begins 2, 4 or 8 bytes behind a 16-byte boundary is moved in narrower pieces."""
    shape = (2, 6, 2, 2, 16, 24)
    for skip in (1, 2, 4):
        buf = torch.randn(2 * 6 * 2 * 2 * 16 * 24 + 8, device="cuda").to(torch.bfloat16)
        x = buf[skip:skip + 2 * 6 * 2 * 2 * 16 * 24].view(shape)
        want, rest = x.clone(), buf[skip + x.numel():].clone()
        want[:, 4, :, :, :7], want[:, 1] = x[:, 0, :, :, :7], x[:, 3]
        K.copy_pages(x, torch.tensor([[0, 4, 7], [3, 1, 16]], dtype=torch.int32))
        assert torch.equal(x, want) and torch.equal(buf[skip + x.numel():], rest)


def test_copy_pages_replayed(K):
    x = torch.randn(2, 8, 2, 2, PAGE, 16, device="cuda")
    plan = torch.tensor([[0, 5, 20], [1, 6, 64]], dtype=torch.int32)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.copy_pages(x, plan)
    plan.zero_()                                          # the recording keeps its own plan
    x[:, 0], x[:, 1] = 3.0, 4.0
    g.replay()
    assert (x[:, 5, :, :, :20] == 3).all() and (x[:, 6] == 4).all() and not (x[:, 5, :, :, 20:] == 3).any()


def test_copy_pages_refusals(K):
    from cima_b200.kernels import KernelError
    x = torch.zeros(1, 4, 1, 1, 4, 8, device="cuda")
    p = lambda *rows: torch.tensor(rows, dtype=torch.int32).view(-1, 3)       # noqa: E731
    for plan, word in [(p([0, 4, 1]), "outside"), (p([-1, 1, 1]), "outside"), (p([0, 1, 5]), "positions"), (p([0, 1, -1]), "positions"),
                       (p([0, 1, 1], [2, 1, 1]), "writes"), (p([0, 1, 1], [1, 2, 1]), "reads"), (p([1, 2, 1], [0, 1, 1]), "writes"), (p([3, 3, 1]), "reads"),
                       (p([0, 1, 1]).cuda(), "host"), (p([0, 1, 1]).long(), "int32")]:
        with pytest.raises(KernelError, match=word):
            K.copy_pages(x, plan)
    with pytest.raises(KernelError, match="contiguous"):
        K.copy_pages(x.transpose(1, 5), p([0, 1, 1]))


# ---------------------------------------------------------------------------------------------- log-probabilities
@pytest.mark.parametrize("n, V", [(1, 1), (1, 2), (3, 7), (1, 512), (5, 1000), (2, 4097), (64, 32003), (1, 151936), (61, 152064), (130, 40000), (700, 5001), (66000, 5), (66000, 1100)])
@pytest.mark.parametrize("spread", [0.0, 3.0, 80.0])
def test_token_logprobs(K, n, V, spread):
    gen = torch.Generator(device="cuda").manual_seed(n + V)
    x = torch.randn(n, V, generator=gen, device="cuda") * spread + 5.0
    t = torch.randint(0, V, (n,), generator=gen, device="cuda", dtype=torch.int32)
    t[::2] = x[::2].argmax(1).int()
    out = torch.full((n,), 9.0, device="cuda")
    K.token_logprobs(x, t, out)
    want, tol = logprob_reference(x, t)
    off = (out.double() - want).abs()
    assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("V", [1023, 1025, 4099, 151937])
def test_token_logprobs_of_rows_at_odd_places(K, V):
    """Rows that begin at any multiple of 4 bytes, and what lies beside them."""
    for skip in (1, 2, 3):
        buf = torch.full((5 * V + 8,), 1e30, device="cuda")
        x = buf[skip:skip + 5 * V].view(5, V)
        x.copy_(torch.randn(5, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(V + skip)))
        t = torch.tensor([0, V - 1, 1, V // 2, V - 2], dtype=torch.int32, device="cuda")
        out = torch.full((5,), 9.0, device="cuda")
        K.token_logprobs(x, t, out)
        want, tol = logprob_reference(x, t)
        assert ((out.double() - want).abs() <= tol).all()


def test_token_logprobs_replayed_and_on_a_stream(K):
    x = torch.randn(9, 30000, device="cuda")
    t = torch.randint(0, 30000, (9,), dtype=torch.int32, device="cuda")
    want = torch.empty(9, device="cuda")
    K.token_logprobs(x, t, want)
    out, side = torch.empty(9, device="cuda"), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.token_logprobs(x, t, out)
    side.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.token_logprobs(x, t, out)
    x.mul_(0.5)
    g.replay()
    K.token_logprobs(x, t, want)
    assert torch.equal(out, want)


def test_token_logprobs_of_infinite_logits(K):
    inf, nan = math.inf, math.nan
    rows = [([0.0, -inf, 1.0], 0, math.log(1 / (1 + math.e))), ([0.0, -inf, 1.0], 1, -inf), ([-inf, -inf, -inf], 1, nan), ([0.0, inf, 1.0], 0, nan),
            ([0.0, inf, 1.0], 1, nan), ([0.0, nan, 1.0], 0, nan), ([nan, nan, nan], 2, nan), ([0.0, 0.0, 0.0], 3, nan), ([0.0, 0.0, 0.0], -1, nan),
            ([3e38, -3e38, 0.0], 0, 0.0), ([3e38, -3e38, 3e38], 0, -math.log(2.0)), ([-inf, 4.0, -inf], 1, 0.0)]
    x = torch.tensor([r[0] for r in rows], device="cuda")
    t = torch.tensor([r[1] for r in rows], dtype=torch.int32, device="cuda")
    out = torch.empty(len(rows), device="cuda")
    K.token_logprobs(x, t, out)
    for got, (_, _, want) in zip(out.tolist(), rows):
        if math.isnan(want):
            assert math.isnan(got)
        else:
            assert got == want or abs(got - want) <= 2.0 ** -21 * abs(want)


def test_token_logprobs_refusals(K):
    from cima_b200.kernels import KernelError
    x, t, o = torch.zeros(3, 5, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.empty(3, device="cuda")
    for args, word in [((x, t[:2], o), "tokens"), ((x, t, o[:2]), "places"), ((x.bfloat16(), t, o), "expected"), ((x, t.long(), o), "expected"),
                       ((x.t(), t, o), "contiguous"), ((x.cpu(), t, o), "GPU")]:
        with pytest.raises(KernelError, match=word):
            K.token_logprobs(*args)
    K.token_logprobs(x[:0], t[:0], o[:0])
