"""Beam search above the step function.

Requests are taken in order, as many at a time as their beams fit the engine's batch and the cache (``plan_beams``).  A
request's prompt runs once, in its first slot; from then on its beams are sequences of the batch, and after every step the
device selects the next beams, rewrites their page tables and moves what they take over from their parents
(kernels/beam.py).  The next step starts from the selected tokens where they lie, before the host has read them; the host
follows one step behind, keeps the ended hypotheses and drops the requests that are done.

A hypothesis ends at a stop token that is among the ``beams`` best continuations of its step (the stop token is not part of
its tokens, but of its score and of the count that its value divides by), after ``max_new_tokens``, or when it holds
``max_seq_len`` positions.

The loop only decides.  It runs steps through a ``stepper`` with ``groups_at_once``, ``open(prompt, length) -> slots``,
``close(slots)``, ``tokens_needed(prompt, length)``, ``prompt(entries, want) -> logits``, ``stack(rows) -> logits``, ``begin(groups)``,
``select(logits, scores, drawn) -> choice``, ``step(slots, choice, groups) -> logits``, ``read(choice)``, ``keep(logits,
groups)`` and ``carry(choice, groups) -> scores``, so that its decisions can be tested without a device.

The reference runs the whole prefix again for every beam and step (src/engine_runtime.cpp:472-569).
"""
from __future__ import annotations

import time
from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from ..sampling import BeamParams
from .generate import GenerationStats


@dataclass
class Hypothesis:
    tokens: List[int] = field(default_factory=list)
    score: float = 0.0               # sum of log-probabilities
    value: float = 0.0               # what hypotheses are ranked by
    finish_reason: str = ""          # "stop", "length" (max_new_tokens), "context" (max_seq_len); "none": no continuation was allowed


def plan_beams(needs: Sequence[int], groups_at_once: int, capacity_tokens: int) -> List[List[int]]:
    """Request indices of each batch, in order: at most ``groups_at_once``, and no more positions than the cache holds."""
    batches: List[List[int]] = []
    held = 0
    for i, need in enumerate(needs):
        if need > capacity_tokens:
            raise ValueError(f"request {i}: the beams' {need} positions do not fit the cache's {capacity_tokens}")
        if not batches or len(batches[-1]) >= groups_at_once or held + need > capacity_tokens:
            batches.append([])
            held = 0
        batches[-1].append(i)
        held += need
    return batches


class _Search:
    """One request's search as the host knows it."""

    def __init__(self, request: int, prompt: Sequence[int], slots: Sequence[int], params: BeamParams, limit: int):
        self.request, self.prompt, self.slots, self.params = request, prompt, list(slots), params
        self.limit = limit                       # most tokens it can draw
        self.parents: List[List[int]] = []       # per selection, by place
        self.tokens: List[List[int]] = []
        self.scores: List[float] = []            # after the last selection
        self.ended: List[Hypothesis] = []        # best value first, at most ``beams``

    def _value(self, score: float, n: int) -> float:
        return score / n ** self.params.length_penalty

    def _path(self, place: int, drawn: int) -> List[int]:
        """The tokens of the sequence that was at ``place`` after ``drawn`` selections."""
        out = []
        for at in range(drawn - 1, -1, -1):
            out.append(self.tokens[at][place])
            place = self.parents[at][place]
        return out[::-1]

    def accept(self, scores, parents, tokens, ended_scores, ended_parents) -> bool:
        """Takes in one selection; True while the search goes on."""
        drawn = len(self.tokens)
        for score, parent in zip(ended_scores, ended_parents):
            if parent >= 0 and score > float("-inf"):
                h = Hypothesis([], score, self._value(score, drawn + 1), "stop")
                # worse than everything in a full list: its tokens need not be read back
                if len(self.ended) < self.params.beams or h.value > self.ended[-1].value:
                    h.tokens = self._path(parent, drawn)
                    self.ended.append(h)
                    self.ended.sort(key=lambda e: -e.value)
                    del self.ended[self.params.beams:]
        self.parents.append(list(parents))
        self.tokens.append(list(tokens))
        self.scores = list(scores)
        drawn += 1
        best = max(self.scores)
        if drawn >= self.limit or best == float("-inf"):
            return False
        if len(self.ended) < self.params.beams:
            return True
        # a running score only falls, and its value is best at the greatest length it can reach
        return not self.params.early_stopping and self._value(best, self.limit) > self.ended[-1].value

    def result(self, max_new: int) -> List[Hypothesis]:
        out = list(self.ended)
        drawn = len(self.tokens)
        if drawn >= self.limit:                  # what still runs has reached its limit
            why = "length" if drawn >= max_new else "context"
            out += [Hypothesis(self._path(p, drawn), s, self._value(s, drawn), why)
                    for p, s in enumerate(self.scores) if s > float("-inf")]
            out.sort(key=lambda h: -h.value)
        # (logits of nothing but -inf and NaN leave no continuation at all)
        return out[:self.params.n_best] or [Hypothesis([], float("-inf"), float("-inf"), "none")]


class BeamLoop:
    def __init__(self, stepper, params: BeamParams, stop_ids: Sequence[int], max_batch: int, max_seq_len: int, capacity_tokens: int,
                 dedicated_prefill: bool = True, prefill_chunk: Optional[int] = None):
        params.check()
        if params.beams > max_batch:
            raise ValueError(f"{params.beams} beams do not fit max_batch {max_batch}")
        if prefill_chunk is not None and prefill_chunk <= 0:
            raise ValueError(f"prefill_chunk must be positive, got {prefill_chunk}")
        self.stepper, self.params = stepper, params
        self.stop_ids = tuple(sorted({int(s) for s in stop_ids}))
        self.max_batch, self.max_seq_len, self.capacity_tokens = max_batch, max_seq_len, capacity_tokens
        self.dedicated_prefill, self.prefill_chunk = dedicated_prefill, prefill_chunk
        self.stats = GenerationStats()

    def run(self, prompts: Sequence[Sequence[int]], max_new: int) -> List[List[Hypothesis]]:
        results: List[List[Hypothesis]] = [[] for _ in prompts]
        todo = []
        for i, p in enumerate(prompts):
            if not len(p):
                raise ValueError(f"request {i}: the prompt is empty")
            if len(p) > self.max_seq_len:
                raise ValueError(f"request {i}: a prompt of {len(p)} tokens exceeds max_seq_len {self.max_seq_len}")
            if max_new <= 0 or len(p) >= self.max_seq_len:
                results[i] = [Hypothesis(finish_reason="length" if max_new <= 0 else "context")]
            else:
                todo.append(i)
        needs = [self.stepper.tokens_needed(len(prompts[i]), min(len(prompts[i]) + max_new, self.max_seq_len)) for i in todo]
        for batch in plan_beams(needs, min(self.max_batch // self.params.beams, self.stepper.groups_at_once), self.capacity_tokens):
            self._run_batch([todo[k] for k in batch], prompts, max_new, results)
        return results

    def _prompts(self, searches: List[_Search]) -> object:
        """Runs the prompts in the groups' first slots; the logits after each, stacked in the searches' order."""
        st = self.stepper
        fed = [0] * len(searches)
        rows: Dict[int, object] = {}
        while len(rows) < len(searches):
            entries, want, whose = [], [], []
            budget = self.prefill_chunk
            for k, s in enumerate(searches):
                left = len(s.prompt) - fed[k]
                n = min(left, 1 if not self.dedicated_prefill else left if budget is None else budget)
                if n <= 0:
                    continue
                if budget is not None:
                    budget -= n
                entries.append((s.slots[0], list(s.prompt[fed[k]:fed[k] + n])))
                fed[k] += n
                want.append([n - 1] if n == left else [])
                if n == left:
                    whose.append(k)
                self.stats.prompt_tokens += n
            got = st.prompt(entries, want)
            for at, k in enumerate(whose):
                rows[k] = (got, at, len(whose))
        return st.stack([rows[k] for k in range(len(searches))])

    def _run_batch(self, batch, prompts, max_new, results) -> None:
        st = self.stepper
        self.stats.batches += 1
        live: List[_Search] = []
        try:
            for i in batch:
                n = len(prompts[i])
                limit = min(max_new, self.max_seq_len - n)
                live.append(_Search(i, prompts[i], st.open(n, n + limit), self.params, limit))
            t0 = time.perf_counter()
            logits = self._prompts(live)
            st.begin([(s.slots, len(s.prompt)) for s in live])
            self.stats.prefill_seconds += time.perf_counter() - t0
            scores = None                        # one beam per request, with probability one
            drawn = 0
            while live:
                t0 = time.perf_counter()
                choice = st.select(logits, scores, drawn)
                drawn += 1
                # the next step starts before this selection is read, unless some request is known to end with it
                ahead = None
                if all(drawn < s.limit for s in live):
                    ahead = st.step([s.slots for s in live], choice, None)
                goes_on = [s.accept(*seen) for s, seen in zip(live, st.read(choice))]
                stays = [k for k, on in enumerate(goes_on) if on]
                for s, on in zip(live, goes_on):
                    if not on:
                        results[s.request] = s.result(max_new)
                        st.close(s.slots)
                        self.stats.generated_tokens += sum(len(h.tokens) for h in results[s.request])
                left = [live[k] for k in stays]
                if left:
                    some = None if len(left) == len(live) else stays
                    logits = st.keep(ahead, some) if ahead is not None else st.step([s.slots for s in left], choice, some)
                    scores = st.carry(choice, some)
                live = left
                self.stats.decode_seconds += time.perf_counter() - t0
                self.stats.decode_steps += 1
        except BaseException:
            for s in live:
                try:
                    st.close(s.slots)
                except Exception:
                    pass
            raise


class BeamStepper:
    """What the loop drives: the engine's steps, the selection, and the cache that follows it."""

    def __init__(self, engine, params: BeamParams, stop_ids: Sequence[int]):
        from ..kernels import beam as KB
        if len(stop_ids) > KB.STOPS_MAX:
            raise ValueError(f"{len(stop_ids)} stop tokens (beam search takes {KB.STOPS_MAX})")
        self.engine, self.beams = engine, params.beams
        # what a cache may not have is found here, not after the prompts have run
        self.groups_at_once = engine.cache.beam_groups(params.beams)
        self.stops = torch.tensor(sorted(stop_ids), dtype=torch.int32, device=engine.device) if len(stop_ids) else None
        self._side = self._host = None
        self._slots = self._lengths = None

    def tokens_needed(self, prompt: int, length: int) -> int:
        return self.engine.cache.beam_tokens(prompt, length, self.beams)

    def open(self, prompt: int, length: int) -> List[int]:
        slots: List[int] = []
        try:
            for _ in range(self.beams):
                slots.append(self.engine.new_sequence())
            self.engine.cache.reserve_beams(slots, prompt, length)
        except BaseException:
            for s in slots:
                self.engine.end_sequence(s)
            raise
        return slots

    def close(self, slots: Sequence[int]) -> None:
        for s in slots:
            self.engine.end_sequence(s)

    def prompt(self, entries, want):
        got = self.engine.step(entries, want)
        return None if got is None else got.clone()      # (a later step may overwrite what a step returns)

    def stack(self, rows) -> torch.Tensor:
        """The logits of one row per group, from (tensor, row, rows of the tensor)."""
        if all(t is rows[0][0] for t, _, _ in rows) and [r for _, r, _ in rows] == list(range(rows[0][2])):
            return rows[0][0]
        return torch.stack([t[r] for t, r, _ in rows])

    def begin(self, groups: Sequence[Tuple[Sequence[int], int]]) -> None:
        for slots, prompt in groups:
            self.engine.cache.begin_beams(slots, prompt)
        self._slots = torch.tensor([list(s) for s, _ in groups], dtype=torch.int32, device=self.engine.device)
        self._lengths = torch.tensor([n for _, n in groups], dtype=torch.int32, device=self.engine.device)

    def select(self, logits: torch.Tensor, scores: Optional[torch.Tensor], drawn: int):
        """Selects, and lets the cache follow; ``drawn``: the tokens that each beam holds behind its prompt."""
        from ..kernels import beam as KB
        with self.engine.tracer.range("beam"):
            if scores is None:
                # (64 bits: a score is a sum over all steps, and 32 would round the whole of it at each)
                scores = torch.zeros(self._slots.shape[0], 1, dtype=torch.float64, device=self.engine.device)
            choice = KB.select(logits, scores, self.beams, self.stops, **({"wide": True} if logits.is_cuda else {}))
            seen = None
            if logits.is_cuda:
                seen = torch.cuda.Event()
                seen.record()
            self.engine.cache.follow_parents(self._slots, choice.parents, self._lengths, drawn)
        return choice, seen

    def _of(self, t: torch.Tensor, groups) -> torch.Tensor:
        return t if groups is None else t[torch.tensor(groups, dtype=torch.long, device=t.device)]

    def step(self, slots, handle, groups) -> torch.Tensor:
        """Every beam of the groups goes on by its token; ``groups``: which of the selection's they are (None: all)."""
        choice, _ = handle
        if groups is not None:
            self._drop(groups)
        flat = [s for of_group in slots for s in of_group]
        ids = self._of(choice.tokens, groups).reshape(-1)
        return self.engine.step([(s, None) for s in flat], [[0] for _ in flat], token_source=ids)

    def keep(self, logits: torch.Tensor, groups) -> torch.Tensor:
        """The rows of a step that was started before some groups were known to be done."""
        if groups is None:
            return logits
        self._drop(groups)
        return self._of(logits.view(-1, self.beams, logits.shape[-1]), groups).reshape(-1, logits.shape[-1])

    def carry(self, handle, groups) -> torch.Tensor:
        """The scores that the next selection starts from."""
        return self._of(handle[0].scores, groups)

    def _drop(self, groups) -> None:
        self._slots, self._lengths = self._of(self._slots, groups), self._of(self._lengths, groups)

    def read(self, handle) -> List[tuple]:
        """Per group what ``_Search.accept`` takes.  On a stream of its own, behind the selection only."""
        choice, seen = handle
        wanted = (choice.scores, choice.parents, choice.tokens, choice.ended_scores, choice.ended_parents)
        if seen is None:
            host = [t.tolist() for t in wanted]
        else:
            n = wanted[0].numel()
            if self._side is None:
                self._side = torch.cuda.Stream(device=choice.scores.device)
            if self._host is None or self._host[0].numel() < n:
                self._host = [torch.empty(n, dtype=t.dtype, pin_memory=True) for t in wanted]
            with torch.cuda.stream(self._side):
                self._side.wait_event(seen)
                for row, t in zip(self._host, wanted):
                    row[:n].copy_(t.view(n), non_blocking=True)
            self._side.synchronize()
            host = [row[:n].view(t.shape).tolist() for row, t in zip(self._host, wanted)]
        return list(zip(*host))
