"""The generation loop: requests in, tokens out, as many batches one after another as it takes.

The loop is host logic only.  It talks to a *stepper* (``ModelStepper`` for a real model; tests use a
scripted one) through four calls: ``open``, ``prefill``, ``decode``, ``close``.  Its decisions follow the
reference's loop for one sequence (src/models/mod.rs:972-1405), applied to every sequence of a batch:

* a prompt that leaves fewer than 16 positions is cut to its first token plus its newest tail
  (:987-1010);
* budget = min(max_tokens, positions - prompt length) (:1145-1147);
* a sampled stop token ends the sequence with reason "stop" and is neither emitted nor counted,
  unless ``ignore_eos`` (:1262-1269); an exhausted budget ends it with reason "length";
* sequences that end leave the batch, the others go on; when all have ended the batch's slots are
  given back and the next batch starts.

Several continuations of a prompt are requests like any other, each with a generator of its own, but the prompt runs once in a
batch: its further sequences are forked from the first and share its pages.
"""
from __future__ import annotations

import time
from dataclasses import dataclass, replace
from typing import Callable, List, Optional, Protocol, Sequence, Union

from ..sampling.options import GenOptions

RESERVED_FOR_ANSWER = 16


@dataclass
class GenResult:
    tokens: List[int]
    finish_reason: str                # "stop" | "length"
    prompt_tokens: int
    truncated: bool = False
    logprobs: Optional[List[float]] = None     # where asked for: of each token, under the model's own distribution (no penalty, temperature or cut)
    stop_logprob: Optional[float] = None       # the same of the stop token that ended the answer and is not among its tokens

    @property
    def logprob(self) -> Optional[float]:
        """Log-probability of the whole answer, its tokens and the stop token that ended it (None where none were asked for)."""
        return None if self.logprobs is None else sum(self.logprobs) + (self.stop_logprob or 0.0)


@dataclass
class GenStats:
    """Counts and times of one ``generate`` call (the reference's GenStats, src/models/transformer.rs:1791-1806)."""
    prompt_tokens: int = 0
    gen_tokens: int = 0
    batches: int = 0
    reused_tokens: int = 0            # prompt tokens that were not run: their keys were still in the cache
    shared_tokens: int = 0            # prompt tokens that were not run: another continuation of the prompt ran them
    prefill_s: float = 0.0
    decode_s: float = 0.0
    decode_steps: int = 0

    @property
    def decode_tok_per_s(self) -> float:
        return self.gen_tokens / self.decode_s if self.decode_s > 0 else 0.0


class Stepper(Protocol):
    """What the loop needs of a stepper.  One that keeps finished sequences for later prompts also has
    ``retain_limit`` (> 0), ``adopt(prompts) -> [(slot | None, tokens in common)]``, ``make_room(needs, slots)``,
    ``retain(slots, histories)`` and takes ``prefill(..., reused=[...])`` (see ``ModelStepper``); the loop uses them
    only when ``retain_limit`` is positive.  One that can fork has ``prefill_copies(slots, prompts, options, copies, reused) -> (slots, tokens)`` and
    ``shared_positions(length)``, the positions of a prompt that a further continuation needs no pages for; one that knows its tokens' log-probabilities takes
    ``logprobs`` (True: wanted) and has ``last_logprobs`` behind every ``prefill`` and ``decode``."""
    max_batch: int                    # most sequences in one batch
    max_position: int                 # most positions a sequence may hold
    cache_tokens: int                 # positions the cache holds in all
    page_size: int

    def open(self, count: int) -> List[int]: ...
    def prefill(self, slots: Sequence[int], prompts: Sequence[Sequence[int]], options: Sequence[GenOptions]) -> List[int]: ...
    def decode(self, slots: Sequence[int], last_tokens: Sequence[int], options: Sequence[GenOptions]) -> List[int]: ...
    def close(self, slots: Sequence[int]) -> None: ...


def fit_prompt(prompt: Sequence[int], max_position: int):
    """(tokens, truncated): the prompt, cut if it would leave fewer than 16 positions."""
    prompt = list(prompt)
    if not prompt:
        raise ValueError("a prompt needs at least one token")
    if len(prompt) + RESERVED_FOR_ANSWER > max_position:
        keep = max(max_position - RESERVED_FOR_ANSWER, 2)
        if keep < len(prompt):
            return [prompt[0]] + prompt[len(prompt) - (keep - 1):], True
    return prompt, False


def continuation(options: GenOptions, k: int) -> GenOptions:
    """The options of a prompt's k-th continuation (from 0): the seed k further on (0, which a generator takes as 1, is left out), and marked as
    the k-th answer, whose generator starts from both mixed (``GenOptions.generator_state``), so that its draws are apart from the others'; the first is what a
    single answer would be."""
    return options if k == 0 else replace(options, seed=(max(options.seed, 1) - 1 + k) % ((1 << 64) - 1) + 1, answer=options.answer + k)


def plan_batches(needs: Sequence[int], max_batch: int, cache_tokens: int, page_size: int, shared: Optional[Sequence[int]] = None) -> List[List[int]]:
    """Requests (by index, in order) packed into batches: at most ``max_batch`` each, and the
    positions each may come to hold (``needs``), rounded up to pages, within the cache.  ``shared[i]`` > 0: request i continues the same prompt
    as request i - 1, and so many positions (whole pages) need no room of their own in one batch with it."""
    batches: List[List[int]] = []
    cur: List[int] = []
    used = 0
    for i, need in enumerate(needs):
        pages = -(-need // page_size) * page_size
        if pages > cache_tokens:
            raise ValueError(f"request {i} may hold {need} positions; the cache holds {cache_tokens}")
        own = pages - (shared[i] if shared is not None and cur else 0)
        if cur and (len(cur) >= max_batch or used + own > cache_tokens):
            batches.append(cur)
            cur, used, own = [], 0, pages
        cur.append(i)
        used += own
    if cur:
        batches.append(cur)
    return batches


class GenerationLoop:
    def __init__(self, stepper: Stepper, eos_ids: Sequence[int] = ()):
        self.stepper = stepper
        self.eos_ids = tuple(eos_ids)
        self.stats = GenStats()
        self._on_token = None

    def generate(self, prompts: Sequence[Sequence[int]],
                 options: Union[GenOptions, Sequence[GenOptions], None] = None,
                 on_token: Optional[Callable[[int, int], None]] = None, continuations: int = 1, logprobs: bool = False) -> List[GenResult]:
        """``on_token(i, token)`` is called for every token of request ``i`` as soon as the step that made it is
        read, in the order of the requests within a step (the reference hands each token's text to its
        ``on_token`` as it is generated, src/models/mod.rs:977, :1307); a stop token is not reported.
        ``continuations`` n > 1: n answers to each prompt (request i n + k is the k-th of prompt i, drawn with ``continuation``'s options), whose prompt
        runs once.  ``logprobs``: the results hold their tokens' log-probabilities."""
        st = self.stepper
        self._on_token = on_token
        copies = int(continuations)
        if copies != continuations or copies < 1:
            raise ValueError(f"{continuations} continuations: at least one, and a whole number")
        if copies > 1 and not hasattr(st, "prefill_copies"):
            raise ValueError("this stepper cannot fork a sequence: one continuation a prompt")
        if logprobs and not hasattr(st, "last_logprobs"):
            raise ValueError("this stepper knows no log-probabilities")
        if hasattr(st, "last_logprobs"):
            st.logprobs = bool(logprobs)
        n = len(prompts)
        if options is None:
            options = GenOptions()
        opts: List[GenOptions] = [options] * n if isinstance(options, GenOptions) else list(options)
        if len(opts) != n:
            raise ValueError(f"{len(opts)} option sets for {n} prompts")
        fitted = [fit_prompt(p, st.max_position) for p in prompts]
        if copies > 1:
            fitted = [f for f in fitted for _ in range(copies)]
            opts = [continuation(o, k) for o in opts for k in range(copies)]
            n *= copies
        budgets = [min(o.max_tokens, st.max_position - len(p)) for (p, _), o in zip(fitted, opts)]
        results: List[Optional[GenResult]] = [None] * n
        self.stats = GenStats()
        # a request with no budget produces nothing and needs no step
        todo = []
        for i in range(n):
            if budgets[i] <= 0:
                results[i] = GenResult([], "length", len(fitted[i][0]), fitted[i][1], [] if logprobs else None)
            else:
                todo.append(i)
        needs = [len(fitted[i][0]) + budgets[i] for i in todo]
        shared = None
        if copies > 1:
            alike = [j > 0 and todo[j] // copies == todo[j - 1] // copies for j in range(len(todo))]
            shared = [st.shared_positions(len(fitted[i][0])) if a else 0 for i, a in zip(todo, alike)]
        for batch in plan_batches(needs, st.max_batch, st.cache_tokens, st.page_size, shared):
            self._run_batch([todo[j] for j in batch], fitted, budgets, opts, results, copies, logprobs)
        return results  # type: ignore[return-value]

    def _run_batch(self, ids, fitted, budgets, opts, results, copies: int = 1, logprobs: bool = False) -> None:
        st = self.stepper
        # the requests whose prompt runs: the first of each prompt's continuations in this batch
        heads = [j for j, i in enumerate(ids) if j == 0 or copies == 1 or i // copies != ids[j - 1] // copies]
        counts = [b - a for a, b in zip(heads, heads[1:] + [len(ids)])]
        prompts = [fitted[i][0] for i in ids]
        lead = [prompts[j] for j in heads]
        # a stepper that keeps finished sequences offers them to prompts that begin alike
        keeps = getattr(st, "retain_limit", 0) > 0
        taken = st.adopt(lead) if keeps else [(None, 0)] * len(lead)
        reused = [n for _, n in taken]
        slots: List[int] = [s for s, _ in taken if s is not None]
        done = False
        try:
            if keeps:
                if copies == 1:
                    needs = [len(p) + budgets[i] for p, i in zip(prompts, ids)]
                    st.make_room(needs, [s for s, _ in taken])
                else:
                    room, at = [], []
                    for j, n, (s, _) in zip(heads, counts, taken):
                        whole = [len(prompts[k]) + budgets[ids[k]] for k in range(j, j + n)]
                        room += whole[:1] + [w - st.shared_positions(len(prompts[j])) for w in whole[1:]]
                        at += [s] + [None] * (n - 1)
                    st.make_room(room, at)
            fresh = iter(st.open(sum(1 for s, _ in taken if s is None)))
            slots = [s if s is not None else next(fresh) for s, _ in taken]
            self.stats.batches += 1
            stops = [set(self.eos_ids) | set(opts[i].stop) for i in ids]
            out: List[List[int]] = [[] for _ in ids]
            lps: List[List[float]] = [[] for _ in ids]
            t0 = time.perf_counter()
            if len(heads) < len(ids):
                slots, tokens = st.prefill_copies(slots, lead, [opts[i] for i in ids], counts, reused=reused)
            elif any(reused):
                tokens = st.prefill(slots, prompts, [opts[i] for i in ids], reused=reused)
            else:
                tokens = st.prefill(slots, prompts, [opts[i] for i in ids])
            self.stats.prefill_s += time.perf_counter() - t0
            self.stats.prompt_tokens += sum(len(p) for p in prompts)
            self.stats.reused_tokens += sum(reused)
            self.stats.shared_tokens += sum((n - 1) * len(p) for n, p in zip(counts, lead))
            live = list(range(len(ids)))
            while True:
                nxt = []
                scores = st.last_logprobs if logprobs else [None] * len(live)
                for j, t, score in zip(live, tokens, scores):
                    i = ids[j]
                    if t in stops[j] and not opts[i].ignore_eos:
                        results[i] = GenResult(out[j], "stop", len(prompts[j]), fitted[i][1], lps[j] if logprobs else None, score)
                        continue
                    out[j].append(int(t))
                    if logprobs:
                        lps[j].append(score)
                    if self._on_token is not None:
                        self._on_token(i, int(t))
                    if len(out[j]) >= budgets[i]:
                        results[i] = GenResult(out[j], "length", len(prompts[j]), fitted[i][1], lps[j] if logprobs else None)
                        continue
                    nxt.append(j)
                live = nxt
                if not live:
                    break
                t0 = time.perf_counter()
                tokens = st.decode([slots[j] for j in live], [out[j][-1] for j in live], [opts[ids[j]] for j in live])
                self.stats.decode_s += time.perf_counter() - t0
                self.stats.decode_steps += 1
            self.stats.gen_tokens += sum(len(o) for o in out)
            if keeps:
                st.retain(slots, [list(p) + o for p, o in zip(prompts, out)])
                done = True
        finally:
            if not done:
                st.close(slots)
