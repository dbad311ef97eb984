"""What a one-token step knows of its sequences' common pages: splits and order of the attention's blocks (no GPU)."""
import pytest

from helpers import TINY, random_tokens
from test_continuations_cpu import _lm
from cima_b200.engine import StepEntry
from cima_b200.engine import model as engine_model
from cima_b200.engine.graph import shared_shape, step_shape
from cima_b200.kernels import shared_splits


def test_a_sequence_alone_beside_uneven_groups_is_not_taken_for_a_shared_one():
    """Groups of 6 and 2 and one sequence alone: as many sequences as two groups of 6 could hold, and yet one shares nothing; its 250 pages are split as
    they are beside even groups."""
    even, uneven = [([0, 1], 250), ([2, 3], 250)], [([0, 1, 2, 3, 4, 5], 250), ([6, 7], 250)]
    assert step_shape(even, 5) == (2, 2, 256, True) and step_shape(even, 4) == (2, 2, 256, False)
    assert step_shape(uneven, 9) == (2, 8, 256, True) and step_shape(uneven, 8) == (2, 8, 256, False) and step_shape([], 8) == ()
    for heads, kv, rows in ((28, 4, 128), (28, 4, 16), (40, 8, 128)):
        own = [shared_splits(n, m, B, heads, kv, 16100, rows, 256, alone)[1] for n, m, B, alone in ((2, 2, 5, True), (2, 8, 9, True), (2, 8, 8, False))]
        assert own[0] == own[1] >= 8 and own[2] < own[1]
    # not told, it goes by the numbers alone
    assert shared_splits(2, 2, 5, 28, 4, 16100) == shared_splits(2, 2, 5, 28, 4, 16100, alone=True)


@pytest.mark.parametrize("extra", [0, 1])
def test_a_step_says_whether_some_sequence_is_alone(monkeypatch, extra):
    monkeypatch.setattr(engine_model, "worth_sharing", lambda groups, *a: bool(groups))
    lm = _lm("B", max_tokens=2048)
    c, V = lm.model.cache, TINY["B"]["vocab_size"]
    slots = []
    for n, seed in ((3, 1), (2, 2)):
        (a,) = c.open(1)
        lm.step([StepEntry(a, random_tokens(V, 70, seed))])
        slots += [a] + c.fork(a, n - 1)
    for _ in range(extra):
        (a,) = c.open(1)
        lm.step([StepEntry(a, random_tokens(V, 90, 3))])
        slots.append(a)
    seen, whole = [], lm.model.forward
    monkeypatch.setattr(lm.model, "forward", lambda batch: (seen.append(batch.shared), whole(batch))[1])
    lm.step([StepEntry(s, [1], [0]) for s in slots])
    (shared,) = seen
    assert shared.alone == bool(extra) and shared.groups.tolist() == [[0, 3, 1], [3, 2, 1]] and shared.most == 4


def _endings(rng, prompts, answers):
    """The plans that a batch of several prompts' answers passes through as they end one after another."""
    left = [answers] * prompts
    while any(left):
        at, groups = 0, []
        for n in left:
            if n > 1:
                groups.append((list(range(at, at + n)), 250))
            at += n
        yield groups, at
        alive = [i for i, n in enumerate(left) if n]
        left[rng.choice(alive)] -= 1


def test_the_shapes_that_answers_pass_through_stay_few():
    import random
    rng = random.Random(1)
    for prompts, answers in ((3, 8), (8, 4), (1, 32)):
        seen, exact = {}, set()
        for _ in range(300):
            for groups, n in _endings(rng, prompts, answers):
                shape = step_shape(groups, n)
                if not groups:
                    assert shape == ()
                    continue
                g, most, pages, alone = shape
                assert len(groups) <= g <= n and max(len(m) for m, _ in groups) <= most <= n and pages == 256
                assert alone == (sum(len(m) for m, _ in groups) < n)
                seen.setdefault(n, set()).add(shape)
                exact.add((n, *shared_shape(groups), alone))
        total = sum(len(s) for s in seen.values())
        assert total <= len(exact) and (prompts == 1) <= (total == answers - 1)
        if prompts > 1:
            assert total < 0.6 * len(exact)


def test_spare_places_of_a_plan_are_groups_without_sequences():
    from cima_b200.cache import SharedPrefixes
    packed = SharedPrefixes.pack([([1, 3], 5)], 4, 3)
    assert packed.tolist() == [1, 3, 0, 2] + [0, 5, 0, 5] + [0, 2, 5] + [0] * 6


def test_recordings_of_sequences_that_share_are_bounded(monkeypatch):
    """So many are kept, the one used longest ago gives way, but not what is armed or in flight; those of sequences that share nothing are kept all."""
    from types import SimpleNamespace
    import torch
    from cima_b200.engine import graph
    lm = _lm("B")
    st = lm.stepper
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(graph, "DecodeGraph", lambda model, sampler, n, greedy, bound, pool, shape, logprobs: SimpleNamespace(key=(n, greedy, bound, shape, logprobs)))
    monkeypatch.setattr(graph, "MAX_SHARED_GRAPHS", 4)
    key = lambda n, shape=(): (n, True, 0, shape, False)                # noqa: E731
    shared = lambda n: key(n, (1, n, 4, False))                         # noqa: E731
    plain = [st._graph(key(n)) for n in range(1, 40)]
    first = st._graph(shared(2))
    assert first.key == shared(2) and st._graph(shared(2)) is first
    flown = st._graph(shared(3))
    st._armed, st._flight = (shared(2), (), []), {"graph": flown}
    for n in range(4, 20):
        assert st._graph(shared(n)).key == shared(n)
        kept = [k for k in st._graphs if k[3]]
        assert len(kept) <= 4 and shared(2) in kept and shared(3) in kept and shared(n) in kept
    assert [k for k in st._graphs if k[3]][-2:] == [shared(18), shared(19)]
    st._armed = st._flight = None
    st._graph(shared(18))
    for n in range(20, 23):
        st._graph(shared(n))
    assert [k for k in st._graphs if k[3]] == [shared(18), shared(20), shared(21), shared(22)]
    assert all(st._graphs[key(n)] is g for n, g in zip(range(1, 40), plain))


def test_no_plan_is_made_where_no_layer_could_read_it(monkeypatch):
    """Head sizes above 128, windows, shared value heads and pages other than 64 take the ordinary kernels: no plan, and no recordings of their own."""
    from cima_b200.parts.attention import Attention
    from cima_b200.parts.diff_attention import DiffAttention
    assert not getattr(DiffAttention, "reads_shared", False)
    monkeypatch.setattr(engine_model, "worth_sharing", lambda groups, *a: bool(groups))

    def groups(lm):
        (a,) = lm.model.cache.open(1)
        lm.step([StepEntry(a, random_tokens(TINY["B"]["vocab_size"], 70, 1))])
        return lm.model.shared_groups([a] + lm.model.cache.fork(a, 2))

    assert groups(_lm("B")) == [([0, 1, 2], 1)]
    lm = _lm("B")
    for block in lm.model.blocks:
        assert isinstance(block.mixer, Attention) and block.mixer.reads_shared
        block.mixer.hd = 144
        assert not block.mixer.reads_shared
    monkeypatch.setattr(Attention, "reads_shared", False)
    assert groups(_lm("B")) == []


def test_the_plan_counts_among_the_bytes_sent(monkeypatch):
    """A recorded step's inputs as they are loaded: tokens, places, lengths and slots, the options, and the plan of what is shared."""
    from types import SimpleNamespace
    from cima_b200.engine import graph
    from cima_b200.sampling import GenOptions
    monkeypatch.setattr(engine_model, "worth_sharing", lambda groups, *a: bool(groups))
    lm = _lm("B", max_tokens=2048)
    st, c = lm.stepper, lm.model.cache
    (a,) = c.open(1)
    lm.step([StepEntry(a, random_tokens(TINY["B"]["vocab_size"], 70, 1))])
    slots = [a] + c.fork(a, 2)

    def recording(model, sampler, n, greedy, bound, pool, shape, logprobs):
        shared = graph.SharedBuffer(shape, n, "cpu") if shape else None
        return SimpleNamespace(load=lambda s, t, lengths, params, groups: shared and shared.load(groups), feed=lambda t: None, shared=shared, max_len=bound)

    monkeypatch.setattr(graph, "DecodeGraph", recording)
    for some, plan in ((slots, 2 * 3 + 3 * 1), (slots[:1], 0)):
        before = st.h2d_bytes
        st._arm(some, [1] * len(some), [GenOptions()] * len(some))
        assert st.h2d_bytes - before == 4 * (6 * len(some) + 1 + 4 * len(some) + plan)


def test_few_sequences_that_may_be_long_have_places_for_their_own_pages():
    """Up to eight sequences over thousands of positions: blocks for long own parts, within what the SMs hold; short contexts and more sequences keep the few."""
    own = lambda n, heads, kv, longest: shared_splits(1, n, n, heads, kv, longest, 128, 96)[1]                # noqa: E731
    for n, heads, kv in ((8, 28, 4), (4, 28, 4), (8, 12, 2), (8, 40, 8)):
        assert min(8, 296 // (n * kv)) == own(n, heads, kv, 14000) and n * kv * own(n, heads, kv, 14000) <= 296
    assert own(8, 28, 4, 900) == 2 and own(16, 28, 4, 14000) == 1 and own(64, 28, 4, 30000) == 1
