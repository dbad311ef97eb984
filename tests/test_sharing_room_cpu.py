"""Sequences that share pages: calls that write nothing take nothing, and groups of any shape are found (no GPU)."""
import pytest

from test_continuations_cpu import Shadow, make
from cima_b200.cache import CacheFull


@pytest.mark.parametrize("length", [1, 63, 64, 65, 100, 128])
def test_reserving_what_is_held_already_takes_nothing(length):
    c = make(pages=3)
    s = Shadow(c)
    (a,) = c.open(1)
    s.held[a] = []
    s.write(a, length)
    (b,) = c.fork(a)
    s.held[b] = list(s.held[a])
    g = c.groups[0]
    before = g.pool.held, g.shared
    for slot in (a, b):
        assert g.written(slot, length, length) == [] and c.shared_tokens(slot, length, length) == 0
        c.reserve(slot, length)
        c.must_fit([(a, length), (b, length)])
    assert (g.pool.held, g.shared) == before and not g.copies
    s.verify()
    (n,) = c.open(1)
    c.reserve(n, c.free_tokens())                        # no page is free: what writes nothing still fits
    c.reserve(b, length)
    c.must_fit([(a, length), (b, length)])
    if length % 64:
        with pytest.raises(CacheFull):
            c.reserve(b, length + 1)
    s.verify()


def test_reserving_at_the_length_in_random_histories():
    import random
    rng = random.Random(3)
    c = make(pages=30, max_seqs=9)
    s = Shadow(c)
    (a,) = c.open(1)
    s.held[a] = []
    for _ in range(200):
        slots = list(s.held)
        a = rng.choice(slots)
        try:
            what = rng.choice(["write", "write", "fork", "close", "rewind"])
            if what == "write":
                s.write(a, rng.choice([1, 5, 63, 64]))
            elif what == "fork":
                for b in c.fork(a, 1):
                    s.held[b] = list(s.held[a])
            elif what == "rewind":
                n = rng.randint(0, len(s.held[a]))
                c.rewind(a, n)
                del s.held[a][n:]
            elif len(slots) > 1:
                c.close([a])
                del s.held[a]
        except CacheFull:
            pass
        held = [(g.pool.held, g.shared, list(g.copies)) for g in c.groups]
        for slot in s.held:
            c.reserve(slot, c.length(slot))
        assert [(g.pool.held, g.shared, list(g.copies)) for g in c.groups] == held
        s.verify()


@pytest.mark.parametrize("n", [40, 1500])
def test_groups_among_sequences_each_forked_from_the_one_before(n):
    """Sequence i holds a page more than the one it was forked from: n prefixes one within the other, and in the comb two leaves at each."""
    from cima_b200.cache import KVCache, KVRequest
    c = KVCache([[KVRequest(1, 1, 0)]], 64 * 3 * n, 64 * (n + 2), __import__("torch").float32, "cpu")
    (a,) = c.open(1)
    chain = []
    for _ in range(n):
        c.reserve(a, c.length(a) + 64)
        c.commit(a, c.length(a) + 64)
        chain.append(a)
        (a,) = c.fork(a)
    # of prefix k (pages), n - k + 1 sequences: (n - k) k pages spared
    (members, pages), = c.shared_groups(chain)
    assert (len(members) - 1) * pages == max((n - k) * k for k in range(1, n)) and sorted(members) == list(range(pages - 1, n))
    # two sequences that end at each length: pairs spare what the whole chain does, and more
    pairs = chain + [c.fork(s)[0] for s in chain[:n // 2]]
    got = c.shared_groups(pairs)
    assert sum((len(m) - 1) * p for m, p in got) >= max((n - k) * k for k in range(1, n))
    assert all(len(set(c.groups[0].table_host[pairs[i], p - 1] for i in m)) == 1 for m, p in got)
    seen = [i for m, _ in got for i in m]
    assert len(seen) == len(set(seen))
