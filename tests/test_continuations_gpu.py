"""Several continuations of a prompt on the GPU: forked pages, attention over the shared prefix and log-probabilities together, as ``LM.generate`` and
``LM.step`` use them."""
import random

import pytest
import torch

import cima_b200
from cima_b200.config.shapes import SHAPES
from cima_b200.engine import StepEntry
from cima_b200.engine.generate import continuation
from cima_b200.sampling import GenOptions

pytestmark = pytest.mark.gpu

_models = {}


def lm_of(shape, dtype, **kw):
    """An LM over a model that tests share (each LM has a stepper of its own)."""
    key = (shape, dtype)
    if key not in _models:
        _models[key] = cima_b200.load(config=SHAPES[shape], seed=3, dtype=dtype, max_tokens=64 * 60, verbose=False).model
    return cima_b200.LM(_models[key], **kw)


@pytest.fixture
def always(monkeypatch):
    """Prefixes are read once however short they are (of these tiny models none would be long enough)."""
    from cima_b200.engine import model
    monkeypatch.setattr(model, "worth_sharing", lambda groups, *a: bool(groups))


def tokens(V, n, seed):
    return [random.Random(seed).randrange(V) for _ in range(1)] + [random.Random(seed * 1000 + i).randrange(V) for i in range(n - 1)]


SMALL = ["tiny-b", "vunovik-tiny", "gisirax-tiny", "lipizen-tiny", "netezen-tiny", "pelatar-tiny", "gudarax-tiny"]


@pytest.mark.parametrize("shape", SMALL)
@pytest.mark.parametrize("pipeline", [True, False])
@pytest.mark.parametrize("opts", [dict(temperature=0, repeat_penalty=1.0), dict(temperature=0.9, top_k=30, seed=9)], ids=["greedy", "sampled"])
def test_continuations_are_what_single_answers_would_be(shape, pipeline, opts, always):
    """32-bit, every architecture (recurrences whose state is copied, rings of windows, layers that read another's keys): each continuation has the
    tokens of a request of its own."""
    lm = lm_of(shape, "float32", pipeline=pipeline)
    V = lm.spec.vocab
    longest = min(150, lm.spec.max_position - 40)
    prompts = [tokens(V, 20, 1), tokens(V, longest, 2)]
    got = lm.generate(prompts, max_tokens=9, ignore_eos=True, continuations=3, logprobs=True, **opts)
    assert lm.stats.shared_tokens == 2 * (20 + longest)
    rest = {a: b for a, b in opts.items() if a != "seed"}
    for i, p in enumerate(prompts):
        for k in range(3):
            o = continuation(GenOptions(max_tokens=9, ignore_eos=True, seed=opts.get("seed", 1)), k)
            (want,) = lm.generate([p], o, logprobs=True, **rest)
            assert got[3 * i + k].tokens == want.tokens
            assert got[3 * i + k].logprobs == pytest.approx(want.logprobs, abs=1e-3)
    lm.model.cache.check()
    assert lm.model.cache.slots.held == 0 and all(g.pool.held == 0 for g in lm.model.cache.groups)


@pytest.mark.parametrize("dtype, near", [("float32", 2e-4), ("bfloat16", 4e-2)])
@pytest.mark.parametrize("shape", ["tiny-b", "vunovik-tiny", "pelatar-tiny", "gudarax-tiny"])
@pytest.mark.parametrize("graphs", [True, False])
def test_steps_of_forks_beside_sequences_of_their_own(shape, dtype, near, graphs, always):
    """Teacher-forced steps of forks, and of the same tokens as sequences that share nothing: the logits agree within what the precision's
    steps may differ from the plain implementation's.  Forks of forks, a rewound one, steps of some of them, other orders."""
    lm = lm_of(shape, dtype, use_graphs=graphs)
    c, V = lm.model.cache, lm.spec.vocab
    base = tokens(V, 140, 5)
    rng = random.Random(6)
    a, = c.open(1)
    lm.step([StepEntry(a, base)])
    live = {a: list(base)}
    for s in c.fork(a, 3):
        live[s] = list(base)
    for step in range(14):
        if step == 4:
            src = sorted(live)[1]
            for s in c.fork(src, 2):
                live[s] = list(live[src])
        if step == 7:
            gone = sorted(live)[0]
            c.close([gone])
            del live[gone]
        if step == 9 and c.can_rewind(sorted(live)[0], 70):
            back = sorted(live)[0]
            c.rewind(back, 70)
            del live[back][70:]
        if step == 10:
            c.compact()
        slots = sorted(live)
        rng.shuffle(slots)
        if step % 5 == 4:
            slots = slots[:-1]
        new = {s: rng.randrange(V) for s in slots}
        got = lm.step([StepEntry(s, [new[s]], [0]) for s in slots])
        for s in slots:
            live[s].append(new[s])
        c.check()
        if step in (0, 3, 5, 8, 9, 11, 13):
            alone = c.open(len(slots))
            lm.step([StepEntry(x, live[s][:-1]) for x, s in zip(alone, slots)])
            want = lm.step([StepEntry(x, [live[s][-1]], [0]) for x, s in zip(alone, slots)])
            c.close(alone)
            assert (got - want).abs().max().item() <= near, step
    c.close(list(live))
    c.check()
    lm.model.check_device()


def test_shared_attention_is_what_runs(monkeypatch, always):
    """A decoding step of continuations with whole pages in common takes the shared kernel, recorded; one without does not."""
    lm = lm_of("tiny-b", "bfloat16", pipeline=False)
    K, calls = lm.model.rt.kernels, []
    whole = K.attention_shared
    monkeypatch.setattr(K, "attention_shared", lambda *a, **kw: (calls.append(a[4].most), whole(*a, **kw))[1])
    lm.generate([tokens(1000, 140, 1)], max_tokens=4, temperature=0, repeat_penalty=1.0, ignore_eos=True, continuations=4)
    assert set(calls) == {4}
    calls.clear()
    lm.generate([tokens(1000, 140, 1), tokens(1000, 140, 2)], max_tokens=4, temperature=0, repeat_penalty=1.0, ignore_eos=True)
    assert not calls


def test_bfloat16_continuations_choose_near_maxima(always):
    """Greedy continuations in bfloat16 equal one another, token by token (their rows hold the same numbers), and so do their log-probabilities."""
    lm = lm_of("tiny-b", "bfloat16")
    got = lm.generate([tokens(1000, 150, 8)], max_tokens=30, temperature=0, repeat_penalty=1.0, ignore_eos=True, continuations=5, logprobs=True)
    assert len({tuple(r.tokens) for r in got}) == 1 and len({tuple(r.logprobs) for r in got}) == 1
    (score,) = lm.score([tokens(1000, 150, 8) + got[0].tokens])
    assert got[0].logprobs == pytest.approx(score[149:], abs=4e-2)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scores_in_pieces(dtype):
    lm = lm_of("tiny-b", dtype)
    seq = tokens(1000, 200, 4)
    a, = lm.model.cache.open(1)
    lg = lm.step([StepEntry(a, seq, list(range(200)))])
    lm.model.cache.close([a])
    want = torch.log_softmax(lg.double(), 1)[torch.arange(199), torch.tensor(seq[1:], device="cuda")].tolist()
    for rows in (256, 64, 33):
        assert lm.score([seq, seq[:3]], rows=rows)[0] == pytest.approx(want, abs=1e-3 if dtype == "float32" else 4e-2)


def test_kept_continuations_and_a_later_turn(always):
    """Kept sequences that share their prompt's pages: the next turn of each goes on from its own, the others' pages stay what they were."""
    lm = lm_of("tiny-b", "float32", retain=4)
    plain = lm_of("tiny-b", "float32")
    p = tokens(1000, 100, 3)
    opts = dict(temperature=0.9, top_k=30, seed=4, max_tokens=8, ignore_eos=True)
    first = lm.generate([p], continuations=4, **opts)
    turns = [p + r.tokens + tokens(1000, 11, 20 + k) for k, r in enumerate(first)]
    got = lm.generate(turns, continuations=2, **opts)
    assert lm.stats.reused_tokens == 4 * (100 + 7)
    lm.model.cache.check()
    lm.stepper.drop_retained()
    assert [r.tokens for r in got] == [r.tokens for r in plain.generate(turns, continuations=2, **opts)]
    lm.model.cache.check()


def test_two_models_caches_on_two_streams(always):
    """Forks of one cache stepped on a side stream while another cache's run on the current one: the results are those of one after the other."""
    lms = [lm_of("tiny-b", "float32"), lm_of("vunovik-tiny", "float32")]
    want = []
    for lm in lms:
        want.append(lm.generate([tokens(500, 140, 1)], max_tokens=6, temperature=0.9, seed=2, ignore_eos=True, continuations=3))
    side = torch.cuda.Stream()
    c = lms[0].model.cache
    with torch.cuda.stream(side):
        got = lms[0].generate([tokens(500, 140, 1)], max_tokens=6, temperature=0.9, seed=2, ignore_eos=True, continuations=3)
    other = lms[1].generate([tokens(500, 140, 1)], max_tokens=6, temperature=0.9, seed=2, ignore_eos=True, continuations=3)
    torch.cuda.synchronize()
    assert [r.tokens for r in got] == [r.tokens for r in want[0]] and [r.tokens for r in other] == [r.tokens for r in want[1]]
    c.check()


def test_wide_heads_and_long_prompts_choose_for_themselves(monkeypatch):
    """A model of the 7B shape's heads (two narrow layers): continuations of a long prompt read it once, recorded and issued, and their logits are those of
    sequences that share nothing; a short prompt's do not."""
    cfg = dict(model_type="qwen2", architectures=["Qwen2ForCausalLM"], num_hidden_layers=2, hidden_size=256, num_attention_heads=28, num_key_value_heads=4, head_dim=128,
               intermediate_size=256, vocab_size=512, rope_theta=1e4, rms_norm_eps=1e-6, tie_word_embeddings=True, max_position_embeddings=8192)
    for graphs in (True, False):
        lm = cima_b200.load(config=cfg, seed=1, dtype="bfloat16", max_tokens=64 * 700, verbose=False, use_graphs=graphs)
        c, K, calls = lm.model.cache, lm.model.rt.kernels, []
        whole = K.attention_shared
        monkeypatch.setattr(K, "attention_shared", lambda *a, **kw: (calls.append(a[4].most), whole(*a, **kw))[1])
        for n, shares in ((6500, True), (200, False)):
            calls.clear()
            base = tokens(512, n, 5)
            a, = c.open(1)
            lm.step([StepEntry(a, base)])
            slots = [a] + c.fork(a, 7)
            hist = [list(base) for _ in slots]
            for step in range(5):
                new = [(7 * i + step) % 512 for i in range(8)]
                got = lm.step([StepEntry(s, [t], [0]) for s, t in zip(slots, new)])
                for h, t in zip(hist, new):
                    h.append(t)
            alone = c.open(2)
            lm.step([StepEntry(s, h[:-1]) for s, h in zip(alone, (hist[2], hist[7]))])
            want = lm.step([StepEntry(s, [h[-1]], [0]) for s, h in zip(alone, (hist[2], hist[7]))])
            assert (got[[2, 7]] - want).abs().max().item() <= 4e-2
            assert (8 in calls) == shares
            c.close(slots + alone)
            c.check()
        lm.model.check_device()
        del lm


def test_the_command_line_gives_several_answers_with_scores(capsys):
    from cima_b200.cli import main
    args = ["run", "--random-shape", "tiny-b", "5", "17", "3", "--max-tokens", "6", "--ignore-eos", "true", "--seed", "4", "--max-seq", "512"]
    assert main(args + ["--continuations", "3", "--logprobs"]) == 0
    lines = capsys.readouterr().out.strip().split("\n")
    assert len(lines) == 3 and len(set(lines)) == 3
    for line in lines:
        ids, lp = line.split("\t")
        assert len(ids.split()) == 6 and float(lp) < 0
    assert main(args) == 0
    assert capsys.readouterr().out.strip() == lines[0].split("\t")[0]
    with pytest.raises(SystemExit, match="at least one"):
        main(args + ["--continuations", "0"])
