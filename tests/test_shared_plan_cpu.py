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
    assert step_shape(uneven, 9) == (2, 6, 256, True) and step_shape(uneven, 8) == (2, 6, 256, False) and step_shape([], 8) == ()
    assert step_shape(uneven, 9)[:3] == shared_shape(uneven)
    for heads, kv, rows in ((28, 4, 128), (28, 4, 16), (40, 8, 128)):
        own = [shared_splits(n, m, B, heads, kv, 16100, rows, 256, alone)[1] for n, m, B, alone in ((2, 2, 5, True), (2, 6, 9, True), (2, 6, 8, False))]
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
    assert shared.alone == bool(extra) and shared.groups.tolist() == [[0, 3, 1], [3, 2, 1]] and shared.most == 3
