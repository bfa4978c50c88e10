"""Beam search above the step function.

The reference generates one continuation of a prompt (src/sampler/mod.rs:269-305).  Here the `beams` likeliest unfinished
continuations of every prompt go on together: a step runs them as rows that share the prompt's pages, one kernel
chooses the likeliest of all their next tokens, and the cache lets each go on from the one it extends.

The decisions are plain Python over numbers and can be followed without a device: `generate_beams` needs an engine with
`start_sequences`, `end_sequences`, `prefill` (or `step`), `step(..., groups=...)`, `fork`, `reorder`, and a `select(logits, scores, n)` that gives
(values, beams, tokens) as nested lists or tensors."""
from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import Callable, List, Optional, Sequence, Tuple

from ..csrc.build import PAGE_TOKENS

PAGE = PAGE_TOKENS
MAX_CANDIDATES = 128     # what one selection gives per prompt


@dataclass
class Hypothesis:
    """One continuation: its tokens (without the stop token), the sum of the log-probabilities of its tokens (and of the stop token),
    that sum divided by their number to the power of the length penalty."""
    tokens: List[int]
    logprob: float
    score: float
    stopped_at_eos: bool


@dataclass
class BeamResult:
    """The best hypotheses of a prompt, best first."""
    hypotheses: List[Hypothesis] = field(default_factory=list)
    prompt_len: int = 0
    steps: int = 0

    @property
    def tokens(self) -> List[int]:
        return self.hypotheses[0].tokens if self.hypotheses else []

    @property
    def stopped_at_eos(self) -> bool:
        return bool(self.hypotheses) and self.hypotheses[0].stopped_at_eos


def held_pages(prompt_len: int, max_tokens: int, beams: int) -> int:
    """Cache pages that a prompt and its beams can come to hold: the prompt's whole pages once, what follows for every beam.  The
    last generated token is never fed back."""
    whole = prompt_len // PAGE
    own = -(-(prompt_len + max(max_tokens - 1, 0) - whole * PAGE) // PAGE)
    return whole + beams * own


def plan_beam_batches(prompt_lens: Sequence[int], max_tokens: int, beams: int, cache_tokens: int, max_slots: int) -> List[List[int]]:
    """Cuts requests, in their order, into batches that the cache holds in any case."""
    if beams > max_slots:
        raise ValueError(f"{beams} beams need as many sequence slots, the cache has {max_slots}")
    batches: List[List[int]] = []
    cur: List[int] = []
    used = 0
    for i, n in enumerate(prompt_lens):
        need = held_pages(n, max_tokens, beams) * PAGE
        if need > cache_tokens:
            raise ValueError(f"request {i}: a prompt of {n} tokens plus {max_tokens} generated tokens in {beams} beams needs "
                             f"{need} cache tokens, the cache holds {cache_tokens}")
        if cur and ((len(cur) + 1) * beams > max_slots or used + need > cache_tokens):
            batches.append(cur)
            cur, used = [], 0
        cur.append(i)
        used += need
    if cur:
        batches.append(cur)
    return batches


def _score(logprob: float, terms: int, penalty: float) -> float:
    return logprob / (terms ** penalty) if terms else logprob


class _Search:
    """The hypotheses and the live beams of one prompt."""

    def __init__(self, beams: int, max_tokens: int, penalty: float, stop: set, early: bool):
        self.beams, self.max_tokens, self.penalty, self.stop, self.early = beams, max_tokens, penalty, stop, early
        self.live: List[Tuple[float, List[int]]] = [(0.0, [])]      # (log-probability, tokens), best first
        self.finished: List[Hypothesis] = []
        self.done = False

    def _finish(self, logprob: float, tokens: List[int], stopped: bool) -> None:
        h = Hypothesis(tokens, logprob, _score(logprob, len(tokens) + (1 if stopped else 0), self.penalty), stopped)
        self.finished.append(h)
        self.finished.sort(key=lambda x: -x.score)       # (stable: of equal ones the earlier stays)
        del self.finished[self.beams:]

    def advance(self, values, beams, tokens) -> List[Tuple[int, int]]:
        """Takes the likeliest continuations in falling order; returns (beam it goes on from, its token) of each live beam."""
        new, going = [], []
        for v, b, t in zip(values, beams, tokens):
            if b < 0 or v == -math.inf:
                break
            if t in self.stop:
                if len(going) < self.beams:      # a stop that is behind all live beams does not count
                    self._finish(v, self.live[b][1], True)
                continue
            if len(going) < self.beams:
                new.append((v, self.live[b][1] + [t]))
                going.append((b, t))
        self.live = new
        terms = len(new[0][1]) if new else 0
        if terms >= self.max_tokens or not new:
            for v, toks in new:
                self._finish(v, toks, False)
            self.done = True
        elif len(self.finished) >= self.beams:
            # a sum of log-probabilities only falls: the best that can still come of a live beam
            most = self.max_tokens if self.penalty > 0 else terms + 1
            self.done = self.early or self.finished[-1].score >= _score(new[0][0], most, self.penalty)
        return [] if self.done else going


def _lists(selected):
    """(values, beams, tokens) as nested lists, in one copy where they are parts of one tensor on the device."""
    return [x.tolist() if hasattr(x, "tolist") else x for x in selected]


def generate_beams(engine, select: Callable, prompts: Sequence[Sequence[int]], max_tokens: int, beams: int = 4,
                   length_penalty: float = 1.0, stop_ids: Sequence[int] = (), n_best: int = 1, early_stop: bool = False,
                   cache_tokens: Optional[int] = None, max_batch: Optional[int] = None, to_lists: Callable = _lists) -> List[BeamResult]:
    """The `n_best` likeliest continuations of up to `max_tokens` tokens of every prompt, as a search of `beams` beams finds them.

    At every step the continuations of all live beams are taken in falling order of their log-probability (of equal ones the lower
    beam, then the lower token): one that ends with a stop token becomes a hypothesis if fewer than `beams` others
    came before it, of the rest the first `beams` go on.  Hypotheses rank by log-probability / terms ** length_penalty.  A search ends when
    no live beam can still get among its best `beams` hypotheses (`early_stop`: when it has `beams`), or at `max_tokens`.
    `max_batch`: sequences (beams of all prompts) of one step."""
    if max_tokens < 0:
        raise ValueError("max_tokens must be >= 0")
    stop = set(int(t) for t in stop_ids)
    if beams < 1 or beams * (1 + len(stop)) > MAX_CANDIDATES:
        raise ValueError(f"beams must be at least 1 and beams * (1 + stop tokens) at most {MAX_CANDIDATES}: "
                         f"got {beams} beams and {len(stop)} stop tokens")
    if not 1 <= n_best <= beams:
        raise ValueError(f"n_best must lie in 1 to {beams}, got {n_best}")
    if not math.isfinite(length_penalty):
        raise ValueError("the length penalty must be a finite number")
    if max_tokens > 1 and abs(length_penalty) * math.log2(max_tokens) > 1000:
        raise ValueError(f"a length penalty of {length_penalty} takes {max_tokens} tokens out of the range of numbers")
    for i, p in enumerate(prompts):
        if len(p) == 0:
            raise ValueError(f"request {i}: the prompt is empty")
    results = [BeamResult(prompt_len=len(p)) for p in prompts]
    if max_tokens == 0 or not prompts:
        return results
    cache_tokens = cache_tokens if cache_tokens is not None else engine.cache.max_tokens
    max_batch = max_batch if max_batch is not None else engine.cache.max_slots
    for batch in plan_beam_batches([len(p) for p in prompts], max_tokens, beams, cache_tokens, max_batch):
        slots = engine.start_sequences(len(batch) * beams)
        held = set(slots)

        def end(ss):
            held.difference_update(ss)
            engine.end_sequences(ss)
        try:
            searches = [_Search(beams, max_tokens, length_penalty, stop, early_stop) for _ in batch]
            rows = [slots[j * beams:(j + 1) * beams] for j in range(len(batch))]       # the slots of each prompt's beams
            feed = getattr(engine, "prefill", None) or (lambda s, p: engine.step(s, p, want="last"))
            logits = feed([r[0] for r in rows], [list(prompts[i]) for i in batch])
            chosen = to_lists(select(logits, [[0.0] for _ in batch], min(beams * (1 + len(stop)), logits.shape[1])))
            going = [s.advance(*(c[j] for c in chosen)) for j, s in enumerate(searches)]
            live = [j for j, s in enumerate(searches) if not s.done]
            if live:
                engine.fork([rows[j][0] for j in live for _ in range(beams - 1)], [r for j in live for r in rows[j][1:]])
            while live:
                tokens, parents, scores = [], [], []
                for k, j in enumerate(live):
                    # a place without a beam (fewer continuations than beams exist) runs along without a score
                    pad = beams - len(going[j])
                    parents += [k * beams + b for b, _ in going[j]] + [k * beams] * pad
                    tokens += [[t] for _, t in going[j]] + [[going[j][0][1]]] * pad
                    scores.append([v for v, _ in searches[j].live] + [-math.inf] * pad)
                    results[batch[j]].steps += 1
                flat = engine.reorder([s for j in live for s in rows[j]], parents)
                for k, j in enumerate(live):
                    rows[j] = flat[k * beams:(k + 1) * beams]
                logits = engine.step(flat, tokens, want="last", groups=[beams] * len(live))
                n = min(beams * (1 + len(stop)), beams * logits.shape[1])
                chosen = to_lists(select(logits, scores, n))
                for k, j in enumerate(live):
                    going[j] = searches[j].advance(*(c[k] for c in chosen))
                for j in [j for j in live if searches[j].done]:
                    end(rows[j])                     # its slots and pages are free at once
                live = [j for j in live if not searches[j].done]
            for i, s in zip(batch, searches):
                results[i].hypotheses = s.finished[:n_best]
        finally:
            if held:
                end(list(held))
    return results
