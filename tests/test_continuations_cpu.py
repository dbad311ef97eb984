"""Sequences that share pages: the cache's bookkeeping, several continuations of a prompt, log-probabilities (no GPU; plain statements of the kernels)."""
import math
import random

import pytest
import torch

from helpers import TINY, cpu_model, model_folder, random_tokens
from qwen2_plain import plain_forward, plain_load
from reference_kernels import ReferenceKernels
from cima_b200.cache import CacheFull, KVCache, KVRequest, SharedPrefixes, StateRequest
from cima_b200.engine import GenerationLoop, StepEntry, plan_batches
from cima_b200.engine.generate import continuation
from cima_b200.sampling import GenOptions


def make(pages=12, window=0, max_seqs=None, sites=1, state=()):
    reqs = [[KVRequest(2, 4, 0)] for _ in range(sites)]
    if window:
        reqs.append([KVRequest(2, 4, window)])
    return KVCache(reqs, 64 * pages, 4096, torch.float32, "cpu", max_seqs=max_seqs, extra_state=state)


class Shadow:
    """What every open slot should hold, beside a cache whose 'kernel' writes a mark at each position."""

    def __init__(self, cache):
        self.c, self.held, self.mark = cache, {}, 0

    def write(self, slot, n):
        c, start = self.c, self.c.length(slot)
        c.reserve(slot, start + n)
        c.flush()
        marks = list(range(self.mark + 1, self.mark + 1 + n))
        self.mark += n
        at = torch.arange(start, start + n)
        for g in c.groups:
            e = at // 64 % g.ring_pages if g.ring_pages else at // 64
            g.storage[:, g.block_table[slot].long()[e], :, :, at % 64] = torch.tensor(marks, dtype=torch.float32).view(-1, 1, 1, 1, 1)
        self.held[slot] += marks
        c.commit(slot, start + n)

    def verify(self):
        self.c.flush()
        self.c.check()
        for slot, marks in self.held.items():
            assert self.c.length(slot) == len(marks)
            for g in self.c.groups:
                first = 0 if not g.ring_pages else max(0, len(marks) - g.request.window)
                at = torch.arange(first, len(marks))
                e = at // 64 % g.ring_pages if g.ring_pages else at // 64
                got = g.storage[:, g.block_table[slot].long()[e], :, :, at % 64]         # [positions, layers, planes, heads, values]
                assert (got == torch.tensor(marks[first:], dtype=torch.float32).view(-1, 1, 1, 1, 1)).all(), slot


@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("seed", range(6))
def test_random_histories_of_slots_that_share(window, seed):
    """Opening, writing, forking (shared and outright), rewinding, trimming, compacting and closing in any order: no sequence ever sees
    another's tokens, and no page is lost."""
    rng = random.Random(seed)
    c = make(pages=30, window=window, max_seqs=9)
    s = Shadow(c)
    for _ in range(220):
        slots = list(s.held)
        what = rng.choice(["open", "write", "write", "write", "write", "fork", "fork", "outright", "rewind", "trim", "compact", "close"])
        try:
            if what == "open":
                (n,) = c.open(1)
                s.held[n] = []
            elif what == "compact":
                c.compact()
                for g in c.groups:
                    assert all(p < g.pool.held for pages in g.pages_of for p in pages)
            elif not slots:
                continue
            elif what == "write":
                s.write(rng.choice(slots), rng.choice([1, 1, 5, 64] if window else [1, 1, 5, 63, 64, 130]))
            elif what in ("fork", "outright"):
                a = rng.choice(slots)
                for b in c.fork(a, rng.randint(0, 3), share=what == "fork"):
                    s.held[b] = list(s.held[a])
            elif what == "rewind":
                a = rng.choice(slots)
                n = rng.randint(0, len(s.held[a]))
                if c.can_rewind(a, n):
                    c.rewind(a, n)
                    del s.held[a][n:]
            elif what == "trim":
                c.trim(rng.choice(slots))
            elif what == "close":
                a = rng.choice(slots)
                c.close([a])
                del s.held[a]
        except CacheFull:
            pass
        s.verify()
    c.close(list(s.held))
    c.check()
    assert all(g.pool.held == 0 and g.shared == 0 for g in c.groups) and c.slots.held == 0


def test_a_fork_takes_no_page_until_it_writes_and_the_last_holder_writes_in_place():
    c = make(pages=8)
    s = Shadow(c)
    (a,) = c.open(1)
    s.held[a] = []
    s.write(a, 100)
    b, d = c.fork(a, 2)
    s.held[b], s.held[d] = list(s.held[a]), list(s.held[a])
    g = c.groups[0]
    assert g.pool.held == 2 and g.shared == 2 and c.free_tokens() == 6 * 64
    c.must_fit([(a, 101), (b, 101), (d, 101)])          # two copies: the third writes into the page itself
    s.write(b, 1)
    assert g.pool.held == 3 and g.holders.tolist().count(2) == 1
    s.write(d, 1)
    assert g.pool.held == 4
    s.write(a, 1)
    assert g.pool.held == 4 and g.shared == 1
    s.verify()
    c.close([a, b])
    assert g.pool.held == 2 and g.shared == 0
    del s.held[a], s.held[b]
    s.verify()


def test_room_is_asked_for_before_a_page_is_taken():
    c = make(pages=5, sites=1, window=70)
    s = Shadow(c)
    (a,) = c.open(1)
    s.held[a] = []
    s.write(a, 64), s.write(a, 64), s.write(a, 10)
    assert [len(g.pages_of[a]) for g in c.groups] == [3, 3] and c.groups[1].ring_pages == 3
    with pytest.raises(CacheFull, match="forked 1 times"):
        c.fork(a)                                        # the ring's pages would have to be copied: three wanted, two free
    assert c.slots.held == 1
    c = make(pages=3)
    s = Shadow(c)
    (a,) = c.open(1)
    s.held[a] = []
    s.write(a, 100)
    (b,) = c.fork(a)
    s.held[b] = list(s.held[a])
    c.must_fit([(a, 101), (b, 101)])
    with pytest.raises(CacheFull):
        c.must_fit([(a, 129), (b, 101)])
    with pytest.raises(CacheFull):
        c.reserve(b, 200)                                # a copy and two pages more
    s.verify()
    s.write(b, 1)
    s.write(a, 28)
    s.verify()
    with pytest.raises(ValueError, match="not open"):
        c.fork(2)
    with pytest.raises(ValueError, match="forked -1"):
        c.fork(a, -1)
    with pytest.raises(CacheFull):
        c.fork(a, 2)                                     # three slots, two held


def test_a_page_copied_from_and_taken_anew_before_the_copies_run():
    """b's copy is pending when its source is given back and becomes the target of another copy: the plans keep the order."""
    c = make(pages=4)
    s = Shadow(c)
    (a,) = c.open(1)
    s.held[a] = []
    s.write(a, 10)
    (b,) = c.fork(a)
    s.held[b] = list(s.held[a])
    c.reserve(b, 11)                                     # pending: page 0 -> 1
    (d,) = c.fork(b)                                     # runs what is pending
    s.held[d] = list(s.held[b])
    c.reserve(d, 11)                                     # pending: 1 -> 2
    c.close([a])
    del s.held[a]
    c.close([b])
    del s.held[b]
    (e,) = c.open(1)
    s.held[e] = []
    (f,) = c.fork(d)
    s.held[f] = list(s.held[d])
    c.reserve(f, 11)
    s.verify()
    g = c.groups[0]
    g.copies = [(0, 1, 5), (2, 3, 5), (1, 2, 5), (3, 0, 64)]
    assert [p.tolist() for p in g.plans()] == [[[0, 1, 5], [2, 3, 5]], [[1, 2, 5], [3, 0, 64]]]


def test_state_goes_with_a_fork():
    c = make(state=(StateRequest("x", (3, 2)), StateRequest("n", (), torch.int32), StateRequest("r", (1,), torch.int64)))
    (a,) = c.open(1)
    c.state["x"][a], c.state["n"][a], c.state["r"][a] = 2.5, 7, 1 << 40
    b, d = c.fork(a, 2)
    for k in (b, d):
        assert (c.state["x"][k] == 2.5).all() and int(c.state["n"][k]) == 7 and int(c.state["r"][k]) == 1 << 40
    c.state["x"][b] = 0.0
    assert (c.state["x"][a] == 2.5).all()


def test_groups_of_a_step():
    c = make(pages=40, max_seqs=20)
    s = Shadow(c)
    (root,) = c.open(1)
    s.held[root] = []
    s.write(root, 64 * 2 + 10)
    x, y = c.fork(root, 2)
    for k in (x, y):
        s.held[k] = list(s.held[root])
    s.write(x, 64 * 3)
    s.write(y, 64 * 5)
    xs, ys = [x] + c.fork(x, 2), [y] + c.fork(y, 1)
    (z,) = c.open(1)
    c.reserve(z, 300); c.commit(z, 300)
    # two pages are common to all five, five to x's three, seven to y's two
    assert sorted((sorted(m), p) for m, p in c.shared_groups(xs + ys + [z])) == [([0, 1, 2], 5), ([3, 4], 7)]
    assert c.shared_groups([xs[0], z, ys[0]]) == [([0, 2], 2)]
    assert c.shared_groups([xs[1], ys[0], xs[2]]) == [([0, 2], 5)]              # five pages spared; all three together would spare four
    assert c.shared_groups([z, xs[0]]) == [] and c.shared_groups([xs[0]]) == []
    from cima_b200.engine.graph import shared_shape
    assert shared_shape([([1, 3, 2], 5), ([4, 0], 2)]) == (2, 3, 8) and shared_shape([([0, 1], 1)]) == (1, 2, 1) and shared_shape([]) == ()
    packed = torch.from_numpy(SharedPrefixes.pack([([1, 3], 5), ([4, 0], 2)], 6))
    sp = SharedPrefixes.over(packed, 6, 2)
    assert sp.order.tolist() == [1, 3, 4, 0, 2, 5] and sp.own_page.tolist() == [2, 5, 0, 5, 2, 0] and sp.groups.tolist() == [[0, 2, 5], [2, 2, 2]]
    # only whole pages below a sequence's next position
    c.rewind(xs[1], 64 * 3 + 1)
    assert sorted((sorted(m), p) for m, p in c.shared_groups(xs)) == [([0, 1, 2], 3)]
    c.close(xs + ys + [z, root])
    assert not c.groups[0].shared and c.shared_groups([0, 1]) == []


def test_batches_count_a_shared_prompt_once():
    assert plan_batches([200, 200, 200], 8, 64 * 8, 64, [0, 128, 128]) == [[0, 1, 2]]
    assert plan_batches([200, 200, 200, 200], 8, 64 * 8, 64, [0, 128, 128, 128]) == [[0, 1, 2], [3]]
    assert plan_batches([200, 200, 200], 8, 64 * 4, 64, [0, 128, 128]) == [[0], [1], [2]]
    assert plan_batches([200, 200], 8, 64 * 4, 64) == [[0], [1]]


def test_seeds_of_continuations():
    seeds = [continuation(GenOptions(seed=s), k).seed for s in (0,) for k in range(4)]
    assert [max(s, 1) for s in seeds] == [1, 2, 3, 4]
    assert [continuation(GenOptions(seed=(1 << 64) - 2), k).seed for k in range(3)] == [(1 << 64) - 2, (1 << 64) - 1, 1]
    assert continuation(GenOptions(seed=5), 0) == GenOptions(seed=5)


class WithLogprobs(ReferenceKernels):
    def token_logprobs(self, logits, tokens, out):
        out.copy_(torch.log_softmax(logits.double(), 1).gather(1, tokens.long()[:, None])[:, 0])


def _lm(name, max_tokens=1024, retain=0, max_batch=64, **kw):
    import cima_b200
    from cima_b200.engine import load_model
    model = load_model(model_folder(name), dtype="float32", max_tokens=max_tokens, device="cpu", kernels=WithLogprobs(), verbose=False, **kw)
    return cima_b200.LM(model, retain=retain, pipeline=False, max_batch=max_batch)


@pytest.mark.parametrize("name", ["A", "B", "C"])
@pytest.mark.parametrize("opts", [dict(temperature=0, repeat_penalty=1.0), dict(temperature=0.9, top_k=20, seed=7)])
def test_continuations_are_what_single_answers_would_be(name, opts):
    """Each continuation has the tokens of a request of its own with its seed (C keeps a ring of pages for its window)."""
    V = TINY[name]["vocab_size"]
    lm = _lm(name)
    prompts = [random_tokens(V, 20, 1), random_tokens(V, 70, 2)]
    seen = []
    got = lm.generate(prompts, max_tokens=5, continuations=3, on_token=lambda i, t: seen.append((i, t)), **opts)
    assert len(got) == 6 and lm.stats.shared_tokens == 2 * (20 + 70) and lm.stats.batches == 1
    for i, p in enumerate(prompts):
        for k in range(3):
            (want,) = lm.generate([p], continuation(GenOptions(max_tokens=5).set("seed", opts.get("seed", 1)), k), **{a: b for a, b in opts.items() if a != "seed"})
            assert got[3 * i + k].tokens == want.tokens and got[3 * i + k].prompt_tokens == len(p)
            assert [t for j, t in seen if j == 3 * i + k] == want.tokens
    if opts["temperature"]:
        assert len({tuple(r.tokens) for r in got[:3]}) > 1
    lm.model.cache.check()
    assert lm.model.cache.slots.held == 0 and all(g.pool.held == 0 for g in lm.model.cache.groups)


def test_continuations_in_more_batches_than_one_and_kept():
    V = TINY["B"]["vocab_size"]
    lm, plain = _lm("B", max_tokens=64 * 9, max_batch=3), _lm("B")
    p = [random_tokens(V, 90, 3), random_tokens(V, 10, 4)]
    opts = dict(temperature=0.9, top_k=20, seed=7, max_tokens=6)
    want = [r.tokens for r in plain.generate(p, continuations=4, **opts)]
    assert [r.tokens for r in lm.generate(p, continuations=4, **opts)] == want
    assert lm.stats.batches == 3
    # finished continuations stay, sharing their prompt's page; the next turn of one goes on from there and copies what it writes over
    lm = _lm("B", max_tokens=64 * 12, retain=3)
    first = lm.generate(p[:1], continuations=3, **opts)
    lm.model.cache.check()
    assert lm.model.cache.slots.held == 3 and lm.model.cache.groups[0].shared == 1
    turn = p[0] + first[1].tokens + random_tokens(V, 9, 5)
    back = p[0][:30] + random_tokens(V, 40, 6)
    got = lm.generate([turn, back], continuations=2, **opts)
    assert lm.stats.reused_tokens == 90 + 5 + 30
    assert [r.tokens for r in got] == [r.tokens for r in plain.generate([turn, back], continuations=2, **opts)]
    lm.model.cache.check()
    lm.stepper.drop_retained()
    lm.model.cache.check()
    assert lm.model.cache.groups[0].pool.held == 0


def test_log_probabilities_of_answers_and_scores():
    V = TINY["B"]["vocab_size"]
    cfg, W = plain_load(model_folder("B"))
    lm = _lm("B")
    p = [random_tokens(V, 20, 1), random_tokens(V, 33, 2)]
    got = lm.generate(p, max_tokens=6, temperature=0.9, top_k=20, seed=7, continuations=2, logprobs=True)
    assert [r.tokens for r in got] == [r.tokens for r in lm.generate(p, max_tokens=6, temperature=0.9, top_k=20, seed=7, continuations=2)]
    for i, r in enumerate(got):
        whole = p[i // 2] + r.tokens
        lp = torch.log_softmax(plain_forward(W, cfg, whole).double(), 1)
        want = [float(lp[k - 1, whole[k]]) for k in range(1, len(whole))]
        assert r.logprobs == pytest.approx(want[len(p[i // 2]) - 1:], abs=1e-3) and r.logprob == pytest.approx(sum(want[len(p[i // 2]) - 1:]), abs=5e-3)
        for rows in (256, 7, 1):
            (score,) = lm.score([whole], rows=rows)
            assert score == pytest.approx(want, abs=1e-3)
    assert lm.score([[3]]) == [[]]
    assert lm.generate(p, max_tokens=2)[0].logprobs is None and lm.generate(p, max_tokens=2)[0].logprob is None
    assert lm.generate(p[:1], max_tokens=0, logprobs=True)[0].logprobs == []
    for bad, word in [(dict(sequences=[[]]), "at least one token"), (dict(sequences=[[1, V]]), "token ids"), (dict(sequences=[[1, 2]], rows=0), "at least one")]:
        with pytest.raises(ValueError, match=word):
            lm.score(**bad)
    assert lm.model.cache.slots.held == 0
    for bad in (0, -1, 1.5):
        with pytest.raises(ValueError, match="continuations"):
            lm.generate(p, continuations=bad)


def test_a_stepper_that_cannot_fork_says_so():
    from test_generation_loop import Scripted
    with pytest.raises(ValueError, match="fork"):
        GenerationLoop(Scripted()).generate([[1]], GenOptions(max_tokens=1), continuations=2)
    with pytest.raises(ValueError, match="log-probabilities"):
        GenerationLoop(Scripted()).generate([[1]], GenOptions(max_tokens=1), logprobs=True)


def test_steps_of_forks_are_their_own():
    """``LM.step`` on forked slots: every sequence's logits are those of its own tokens; a fork of a fork too."""
    cfg, W = plain_load(model_folder("B"))
    V = cfg["vocab_size"]
    lm = _lm("B")
    c = lm.model.cache
    (a,) = c.open(1)
    base = random_tokens(V, 130, 1)
    lm.step([StepEntry(a, base)])
    b, d = c.fork(a, 2)
    hist = {a: list(base), b: list(base), d: list(base)}
    rng = random.Random(4)
    for step in range(5):
        if step == 2:
            (e,) = c.fork(b)
            hist[e] = list(hist[b])
        entries = []
        for s in hist:
            t = rng.randrange(V)
            hist[s].append(t)
            entries.append(StepEntry(s, [t], [0]))
        lg = lm.step(entries)
        c.check()
        for s, row in zip(hist, lg):
            assert torch.allclose(row, plain_forward(W, cfg, hist[s]).float()[-1], atol=2e-4, rtol=1e-4)
    c.close(list(hist))
    c.check()


def test_prefixes_are_read_once_where_that_is_worth_it():
    from cima_b200.engine.model import worth_sharing
    page = 2 * 4 * 64 * 128 * 2                           # the 7B shape's, bfloat16
    group = lambda n, pages: [(list(range(n)), pages)]   # noqa: E731
    for n, no, yes in ((4, 64, 256), (8, 32, 128), (48, 7, 32)):
        assert not worth_sharing(group(n, no), n, page, False) and worth_sharing(group(n, yes), n, page, False)
    small = 2 * 2 * 64 * 64 * 4
    assert not worth_sharing(group(2, 1), 2, small, True) and worth_sharing(group(2, 4), 2, small, True)
    assert not worth_sharing([], 8, page, False)
