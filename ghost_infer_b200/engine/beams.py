"""Beam search above the decode runner: every sequence goes on as several beams.

The reference samples one continuation (src/main.rs:702-786).  Here a prompt is read once, its slot is forked into as many as
there are beams (pages are shared, see `SequenceCache.fork`), and every step is: one token for all beams of all sequences, the
2 x beams (or more) best of beams x vocabulary (`ops.beam_select`), the ones among them that end the sequence set aside, the others'
first `beams` fed next after the cache has followed them (`SequenceCache.reorder`).  Twice as many candidates as beams leave
enough that do not end: a beam has a candidate that ends for each of the stop tokens.  More stop tokens ask for more candidates, as
many as `ops.beam_select` gives (64); where all of those were ends, fewer beams would go on.  The end of a search goes by log
probability, not by the score that orders results: the score of a beam that goes on still changes with its length.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Sequence

import torch

from ..cache.pages import CacheFullError, pages_for
from ..kernels import ops
from .step import StepEntry

MAX_BEAMS = ops.MAX_BEAM_WIDTH // 2


@dataclass
class BeamResult:
    tokens: List[int]
    log_prob: float                # sum of the tokens' log probabilities, the stop token's among them
    score: float                   # log_prob / (number of tokens) ** length_penalty: what results are ordered by
    finish_reason: str             # "stop", "length" or "capacity"


@dataclass
class _Search:
    """One sequence's beams."""
    slots: List[int]
    tokens: List[List[int]]
    scores: List[float]
    done: List[BeamResult] = field(default_factory=list)
    next_parents: List[int] = field(default_factory=list)


class BeamSearch:
    def __init__(self, engine, beams: int, stop_token_ids: Sequence[int] = (), length_penalty: float = 1.0, batch_size: int = 1):
        if not 1 <= beams <= MAX_BEAMS:
            raise ValueError(f"{beams} beams: 1 to {MAX_BEAMS} are supported")
        if batch_size < 1:
            raise ValueError("batch_size must be at least 1")
        self.engine, self.beams, self.penalty, self.batch_size = engine, beams, float(length_penalty), batch_size
        self.stop = frozenset(int(t) for t in stop_token_ids)
        # a beam's candidates that end the sequence: at most one for each stop token
        self.width = min(beams * (1 + max(1, len(self.stop))), ops.MAX_BEAM_WIDTH)

    def run(self, prompts: Sequence[Sequence[int]], max_new: int) -> List[List[BeamResult]]:
        """For every prompt its best `beams` results, best first."""
        cache = self.engine.cache
        for i, p in enumerate(prompts):
            if len(p) == 0:
                raise ValueError(f"request {i}: empty prompt")
            if len(p) >= cache.max_seq_len:
                raise ValueError(f"request {i}: prompt does not fit: {len(p)} tokens >= context {cache.max_seq_len}")
        out: List[List[BeamResult]] = []
        while len(out) < len(prompts):
            first, n, free = len(out), 0, cache.free_pages
            while n < self.batch_size and first + n < len(prompts):
                need = pages_for(len(prompts[first + n])) + self.beams            # the shared prompt, a page of its own for each beam
                if need > free or (n + 1) * self.beams > cache.slots.free_slots:
                    break
                free -= need
                n += 1
            if n == 0:
                raise CacheFullError(f"request {first} does not fit: a prompt of {len(prompts[first])} tokens and {self.beams} beams")
            out += self._run_batch([list(p) for p in prompts[first:first + n]], max_new)
        return out

    def _score(self, log_prob: float, tokens: int) -> float:
        return log_prob / max(1, tokens) ** self.penalty

    def _run_batch(self, prompts: List[List[int]], max_new: int) -> List[List[BeamResult]]:
        engine, cache, k = self.engine, self.engine.cache, self.beams
        opened: List[int] = []
        try:
            for _ in prompts:
                opened.append(cache.open_slot())
            if max_new <= 0:
                return [[BeamResult([], 0.0, 0.0, "length")] for _ in prompts]
            firsts = list(opened)
            logits = engine.step([StepEntry(s, p, [len(p) - 1]) for s, p in zip(firsts, prompts)])
            searches: List[_Search] = []
            for s in firsts:
                slots = [s]
                for _ in range(k - 1):
                    slots.append(cache.fork(s))
                    opened.append(slots[-1])
                searches.append(_Search(slots, [[]], [0.0]))
            # after the prompt there is one beam a sequence
            live = list(searches)
            scores = torch.zeros((len(live), 1), dtype=torch.float32, device=logits.device)
            runner = None
            while True:
                vocab = logits.shape[1]
                picked = ops.beam_select(logits, scores, min(self.width, scores.shape[1] * vocab))
                values, parents, tokens = (t.cpu().tolist() for t in picked)
                going = []
                for r, search in enumerate(live):
                    if self._advance(search, values[r], parents[r], tokens[r], max_new, cache):
                        going.append((search, search.next_parents))
                live = [s for s, _ in going]
                if not live:
                    break
                cache.reorder([s.slots for s in live], [p for _, p in going])
                order = [slot for s in live for slot in s.slots]
                if runner is None or runner.slots != order:
                    runner = engine.decoder(order)
                try:
                    logits = runner.forward(tokens=[t[-1] for s in live for t in s.tokens])
                except CacheFullError:
                    for s in live:
                        self._end(s, "capacity")
                    break
                scores = torch.tensor([s.scores for s in live], dtype=torch.float32).to(logits.device)
            return [sorted(s.done, key=lambda b: -b.score)[:k] for s in searches]
        finally:
            for s in opened:
                cache.close_slot(s)

    def _end(self, search: _Search, reason: str) -> None:
        for tokens, log_prob in zip(search.tokens, search.scores):
            if log_prob > float("-inf"):
                search.done.append(BeamResult(list(tokens), log_prob, self._score(log_prob, len(tokens)), reason))

    def _advance(self, search: _Search, values, parents, tokens, max_new: int, cache) -> bool:
        """The beams' next tokens; False when the search has ended."""
        k = self.beams
        nxt = []                                      # (log probability, parent, token)
        for rank, (value, parent, token) in enumerate(zip(values, parents, tokens)):
            if parent < 0 or len(nxt) == k:
                break
            if token in self.stop:
                if rank < k:                          # an ending counts only among the best: else it would displace a better beam
                    n = len(search.tokens[parent]) + 1
                    search.done.append(BeamResult(list(search.tokens[parent]), value, self._score(value, n), "stop"))
            else:
                nxt.append((value, parent, token))
        if not nxt:
            return False
        # fewer candidates than beams (a small vocabulary): the last one's slot stands in for those that are missing
        search.next_parents = [p for _, p, _ in nxt] + [nxt[-1][1]] * (k - len(nxt))
        search.tokens = [search.tokens[p] + [t] for _, p, t in nxt] + [search.tokens[nxt[-1][1]] + [nxt[-1][2]]] * (k - len(nxt))
        search.scores = [v for v, _, _ in nxt] + [float("-inf")] * (k - len(nxt))
        if len(search.done) >= k and max(search.scores) <= min(sorted((b.log_prob for b in search.done), reverse=True)[:k]):
            return False                              # nothing that is still going is, or becomes, more probable than they are
        if len(search.tokens[0]) >= max_new:
            self._end(search, "length")
            return False
        if cache.length(search.slots[0]) + 1 > cache.max_seq_len:
            self._end(search, "capacity")
            return False
        return True
