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
