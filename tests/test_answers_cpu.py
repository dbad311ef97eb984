"""Several answers to one prompt: how they are drawn and scored (no GPU)."""
import random

import pytest
import torch

from helpers import TINY, model_folder, random_tokens
from qwen2_plain import plain_forward, plain_load
from test_continuations_cpu import _lm
from cima_b200.engine.generate import continuation
from cima_b200.sampling import GenOptions


def first_draw(state):
    x = state
    x ^= x >> 12
    x = (x ^ x << 25) & (1 << 64) - 1
    x ^= x >> 27
    return (x * 0x2545F4914F6CDD1D & (1 << 64) - 1) / 2.0 ** 64


def test_first_draws_of_answers_are_spread_like_independent_ones():
    """Over 20,000 seeds: two answers of a prompt (neighbours, or the first and another), and the same answer under neighbouring seeds, draw within 0.02 of
    each other as often as independent numbers (1 - 0.98^2), and eight answers among ten equal tokens give as many different ones (10 (1 - 0.9^8)):
    within five standard errors."""
    rng = random.Random(5)
    near = {"next": 0, "first": 0, "seed": 0}
    n, kinds, squares = 20000, 0, 0
    for i in range(n):
        o = GenOptions(seed=rng.getrandbits(63) if i % 2 else i + 1)
        u = [first_draw(continuation(o, k).generator_state) for k in range(8)]
        k = 1 + i % 6
        near["next"] += abs(u[k] - u[k + 1]) < 0.02
        near["first"] += abs(u[0] - u[k]) < 0.02
        near["seed"] += abs(u[k] - first_draw(continuation(GenOptions(seed=o.seed + 1), k).generator_state)) < 0.02
        d = len({int(10 * x) for x in u})
        kinds, squares = kinds + d, squares + d * d
    p = 1 - 0.98 ** 2
    for what, count in near.items():
        assert abs(count / n - p) <= 5 * (p * (1 - p) / n) ** 0.5, what
    spread = (squares / n - (kinds / n) ** 2) ** 0.5
    assert abs(kinds / n - 10 * (1 - 0.9 ** 8)) <= 5 * spread / n ** 0.5


def test_states_of_generators():
    """A request of its own starts from its seed; answers, and the same answers under other seeds, from states of their own, never 0."""
    assert GenOptions(seed=0).generator_state == 1 and GenOptions(seed=(1 << 64) - 1).generator_state == (1 << 64) - 1
    states = [continuation(GenOptions(seed=s), k).generator_state for s in range(1, 65) for k in range(64)]
    assert len(set(states)) == len(states) and min(states) > 0 and max(states) < 1 << 64
    assert continuation(continuation(GenOptions(seed=5), 2), 3) == continuation(GenOptions(seed=5), 5)
    assert GenOptions(seed=7).generator_state == 7


def test_the_sampler_starts_from_them():
    lm = _lm("B")
    options = [continuation(GenOptions(seed=9), k) for k in range(3)]
    lm.stepper.sampler.begin([0, 1, 2], [[1], [2], [3]], options)
    got = [int(x) & (1 << 64) - 1 for x in lm.model.cache.state["sampler.rng"][:3, 0]]
    assert got == [o.generator_state for o in options] and got[0] == 9


def _score(prompt, tokens):
    cfg, W = plain_load(model_folder("B"))
    whole = prompt + tokens
    lp = torch.log_softmax(plain_forward(W, cfg, whole).double(), 1)
    return [float(lp[k - 1, whole[k]]) for k in range(len(prompt), len(whole))]


@pytest.mark.parametrize("after", [0, 1, 3])
def test_an_answer_that_stops_is_scored_with_its_stop_token(after):
    """Its log-probability is that of its tokens and the stop token, which it does not hold; one that stops at once is scored by that alone."""
    lm, p = _lm("B"), random_tokens(TINY["B"]["vocab_size"], 20, 1)
    opts = dict(max_tokens=6, temperature=0, repeat_penalty=1.0, logprobs=True)
    (free,) = lm.generate([p], ignore_eos=True, **opts)
    stop = free.tokens[after]
    want = _score(p, free.tokens[:after + 1])
    assert stop not in free.tokens[:after]
    for n in (1, 3):
        for r in lm.generate([p], stop=stop, continuations=n, **opts):
            assert r.finish_reason == "stop" and r.tokens == free.tokens[:after]
            assert r.logprobs == pytest.approx(want[:-1], abs=1e-3) and r.stop_logprob == pytest.approx(want[-1], abs=1e-3)
            assert r.logprob == pytest.approx(sum(want), abs=5e-3) and r.logprob < 0
    assert free.finish_reason == "length" and free.stop_logprob is None and free.logprob == pytest.approx(sum(free.logprobs))
    (r,) = lm.generate([p], stop=stop, max_tokens=6, temperature=0, repeat_penalty=1.0)
    assert r.finish_reason == "stop" and r.logprobs is None and r.stop_logprob is None and r.logprob is None
