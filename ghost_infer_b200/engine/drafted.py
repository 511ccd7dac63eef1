"""Greedy generation with drafted tokens: several tokens a step where a guess at the next ones is right.

A drafter guesses, from a sequence's tokens so far, how it may go on: a tree of tokens.  One step runs the whole tree
(`Engine.step_tree`), the model's own picks say how far it goes along (`Engine.commit_tree`), and what comes out is what
one-token steps would have picked.  The decisions about ends are the reference's loop's (src/main.rs:766-786), token by token.
"""
from __future__ import annotations

import time
from dataclasses import dataclass
from typing import Callable, Dict, List, Sequence, Tuple

from ..cache.pages import CacheFullError, pages_for
from ..kernels import ops
from .generate import GenerationResult, GenerationStats
from .step import MAX_TREE_NODES, StepEntry, TreeEntry

MAX_SEQS = 1024                # sequences of one step over trees (the tree attention's limit)

# (tokens so far, most nodes) -> (tokens, parents): parents index the returned tokens, -1 continues the last token so far
Drafter = Callable[[Sequence[int], int], Tuple[List[int], List[int]]]


@dataclass
class PromptLookup:
    """Drafts what followed the sequence's last few tokens where they occurred before in it: no model, no training.  Of the latest
    `branches` places where the longest suffix (up to `longest` tokens) occurred, what follows is merged into one tree."""
    longest: int = 3
    branches: int = 3
    length: int = 8

    def __call__(self, tokens: Sequence[int], most: int) -> Tuple[List[int], List[int]]:
        tokens = list(tokens)
        out: List[int] = []
        parents: List[int] = []
        children: Dict[Tuple[int, int], int] = {}
        for n in range(min(self.longest, len(tokens) - 1), 0, -1):
            suffix, found = tokens[-n:], 0
            for at in range(len(tokens) - n - 1, -1, -1):
                if tokens[at + n - 1] != suffix[-1] or tokens[at:at + n] != suffix:
                    continue
                node = -1
                for t in tokens[at + n:at + n + self.length]:
                    child = children.get((node, t))
                    if child is None:
                        if len(out) >= most:
                            break
                        child = children[(node, t)] = len(out)
                        out.append(t)
                        parents.append(node)
                    node = child
                found += 1
                if found == self.branches or len(out) >= most:
                    break
            if out:
                break
        return out, parents


class DraftedLoop:
    def __init__(self, engine, drafter: Drafter, stop_token_ids: Sequence[int] = (), batch_size: int = 8, max_nodes: int = 32):
        if batch_size < 1:
            raise ValueError("batch_size must be at least 1")
        if not 1 <= max_nodes <= MAX_TREE_NODES:
            raise ValueError(f"trees of {max_nodes} nodes: 1 to {MAX_TREE_NODES} are supported")
        if not engine.takes_trees():
            raise ValueError("this model cannot step over trees of drafted tokens")
        self.engine, self.drafter, self.batch_size, self.max_nodes = engine, drafter, batch_size, max_nodes
        self.stop = frozenset(int(t) for t in stop_token_ids)
        self.stats = GenerationStats()

    def run(self, prompts: Sequence[Sequence[int]], max_new: int) -> List[GenerationResult]:
        cache = self.engine.cache
        for i, p in enumerate(prompts):
            if len(p) == 0:
                raise ValueError(f"request {i}: empty prompt")
            if len(p) >= cache.max_seq_len:
                raise ValueError(f"request {i}: prompt does not fit: {len(p)} tokens >= context {cache.max_seq_len}")
        results = [GenerationResult(prompt_tokens=len(p)) for p in prompts]
        first = 0
        while first < len(prompts):
            free, n = cache.free_pages, 0
            while n < min(self.batch_size, MAX_SEQS) and first + n < len(prompts) and n < cache.slots.free_slots:
                need = pages_for(len(prompts[first + n]) + 1)
                if need > free:
                    break
                free -= need
                n += 1
            if n == 0:
                raise CacheFullError(f"request {first} does not fit: its prompt of {len(prompts[first])} tokens needs more pages than are free")
            self._run_batch(prompts, results, list(range(first, first + n)), max_new)
            first += n
        return results

    def _take(self, res: GenerationResult, token: int, length: int, max_new: int) -> bool:
        """One picked token, with `length` tokens cached before it; whether the sequence goes on."""
        if length >= self.engine.cache.max_seq_len:
            res.finish_reason = "capacity"
            return False
        self.stats.gen_tokens += 1
        if token in self.stop:
            res.finish_reason, res.stopped_on = "stop", token
            return False
        res.tokens.append(token)
        if len(res.tokens) >= max_new:
            res.finish_reason = "length"
            return False
        return True

    def _tree(self, slot: int, tokens: List[int], room: int) -> TreeEntry:
        """The sequence's last token and what is drafted behind it, at most `room` nodes in all."""
        drafted, parents = self.drafter(tokens, room - 1) if room > 1 else ([], [])
        drafted, parents = list(drafted)[:room - 1], list(parents)[:room - 1]
        return TreeEntry(slot, [tokens[-1]] + drafted, [-1] + [p + 1 for p in parents])

    def _run_batch(self, prompts, results, ids: List[int], max_new: int) -> None:
        engine, cache = self.engine, self.engine.cache
        slots: Dict[int, int] = {}
        self.stats.batches += 1
        t0, t1 = time.perf_counter(), None
        try:
            for i in ids:
                slots[i] = cache.open_slot()
            if max_new <= 0:
                for i in ids:
                    results[i].finish_reason = "length"
                return
            logits = engine.step([StepEntry(slots[i], prompts[i], [len(prompts[i]) - 1]) for i in ids])
            self.stats.steps += 1
            self.stats.prompt_tokens += sum(len(prompts[i]) for i in ids)
            live = [i for i, t in zip(ids, ops.sample(logits, 0.0, 0, 1.0).cpu().tolist())
                    if self._take(results[i], t, cache.length(slots[i]), max_new)]
            t1 = time.perf_counter()                   # (the picks have been read back: the prompts are through)
            self.stats.prompt_secs += t1 - t0
            while live:
                entries = []
                for i in live:
                    room = min(self.max_nodes, cache.max_seq_len - cache.length(slots[i]), max_new - len(results[i].tokens))
                    entries.append(self._tree(slots[i], list(prompts[i]) + results[i].tokens, room))
                try:
                    step = engine.step_tree(entries)
                except CacheFullError:
                    # no room for the drafts: their first nodes alone, what a one-token step would take
                    entries = [TreeEntry(e.slot, e.tokens[:1], e.parents[:1]) for e in entries]
                    try:
                        step = engine.step_tree(entries)
                    except CacheFullError:
                        for i in live:
                            results[i].finish_reason = "capacity"
                        break
                self.stats.steps += 1
                before = {i: cache.length(slots[i]) for i in live}
                accepted = engine.commit_tree(step, ops.sample(step.logits, 0.0, 0, 1.0))
                going = []
                for i, tokens in zip(live, accepted):
                    on = True
                    for n, t in enumerate(tokens):
                        on = self._take(results[i], t, before[i] + 1 + n, max_new)
                        if not on:
                            break
                    if on:
                        going.append(i)
                live = going
        finally:
            if t1 is not None:
                self.stats.gen_secs += time.perf_counter() - t1
            for s in slots.values():
                cache.close_slot(s)
