"""Several answers to one prompt on the GPU: scores of answers that stop, recorded steps that stay few, steps of groups that are uneven."""
import pytest
import torch

from test_continuations_gpu import always, lm_of, tokens  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pipeline", [True, False])
@pytest.mark.parametrize("after", [0, 1, 3])
def test_an_answer_that_stops_is_scored_with_its_stop_token(pipeline, after, always):
    lm = lm_of("tiny-b", "float32", pipeline=pipeline)
    p = tokens(1000, 140, 1)
    opts = dict(max_tokens=8, temperature=0, repeat_penalty=1.0, logprobs=True)
    (free,) = lm.generate([p], ignore_eos=True, **opts)
    stop = free.tokens[after]
    assert stop not in free.tokens[:after]
    want = lm.score([p + free.tokens[:after + 1]])[0][139:]
    for n in (1, 3):
        for r in lm.generate([p], stop=stop, continuations=n, **opts):
            assert r.finish_reason == "stop" and r.tokens == free.tokens[:after]
            assert r.logprobs == pytest.approx(want[:-1], abs=1e-3) and r.stop_logprob == pytest.approx(want[-1], abs=1e-3)
            assert r.logprob == pytest.approx(sum(want), abs=1e-2) and r.logprob < 0


@pytest.mark.parametrize("pipeline", [True, False])
def test_recordings_that_give_way(pipeline, always, monkeypatch):
    """Answers of three prompts that end one after another, with room for many recordings and for two: the same tokens and scores, and no more than two are
    kept of steps that share."""
    from cima_b200.engine import graph
    from cima_b200.sampling import GenOptions
    prompts = [tokens(1000, n, n) for n in (140, 200, 70)]
    opts = [GenOptions(temperature=0.9, top_k=30, seed=5, max_tokens=n, ignore_eos=True) for n in (7, 5, 9)]
    many = lm_of("tiny-b", "float32", pipeline=pipeline)
    want = [many.generate(prompts, opts, continuations=k, logprobs=True) for k in (4, 3, 4)]
    monkeypatch.setattr(graph, "MAX_SHARED_GRAPHS", 2)
    few = lm_of("tiny-b", "float32", pipeline=pipeline)
    for k, w in zip((4, 3, 4), want):
        got = few.generate(prompts, opts, continuations=k, logprobs=True)
        assert [(r.tokens, r.logprobs) for r in got] == [(r.tokens, r.logprobs) for r in w]
        assert sum(1 for key in few.stepper._graphs if key[3]) <= 2
    assert sum(1 for key in many.stepper._graphs if key[3]) > 2
    few.model.check_device()


def test_uneven_groups_beside_sequences_alone(always):
    """Three answers, two, and two prompts of one: what each would be by itself, recorded and issued."""
    from cima_b200.engine import StepEntry
    for graphs in (True, False):
        lm = lm_of("tiny-b", "float32", use_graphs=graphs)
        c = lm.model.cache
        slots, hist = [], []
        for n, length, seed in ((5, 150, 1), (2, 80, 2), (1, 230, 3), (1, 64, 4)):
            (a,) = c.open(1)
            lm.step([StepEntry(a, tokens(1000, length, seed))])
            new = [a] + c.fork(a, n - 1)
            slots += new
            hist += [tokens(1000, length, seed) for _ in new]
        for step in range(4):
            new = [(37 * i + step) % 1000 for i in range(len(slots))]
            got = lm.step([StepEntry(s, [t], [0]) for s, t in zip(slots, new)])
            for h, t in zip(hist, new):
                h.append(t)
        alone = c.open(len(slots))
        lm.step([StepEntry(x, h[:-1]) for x, h in zip(alone, hist)])
        want = lm.step([StepEntry(x, [h[-1]], [0]) for x, h in zip(alone, hist)])
        assert (got - want).abs().max().item() <= 2e-4
        c.close(slots + alone)
        c.check()
