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
