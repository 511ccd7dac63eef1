"""Several continuations of one sequence, on the host: shared pages, forked and reordered slots, trees, what is refused (no GPU)."""
import random

import numpy as np
import pytest
import torch

from ghost_infer_b200 import cli
from ghost_infer_b200.cache import PAGE_TOKENS, CacheFullError, CacheRequest, PagePool, SequenceCache, StateRequest, pages_for
from ghost_infer_b200.engine.beams import BeamSearch, _Search
from ghost_infer_b200.engine.drafted import DraftedLoop, PromptLookup
from ghost_infer_b200.engine.step import tree_facts
from ghost_infer_b200.kernels import ops
from ghost_infer_b200.kernels.library import KernelError
from branch_cases import ancestors, plain_walk, random_tree


def test_a_page_goes_back_with_its_last_holder():
    pool = PagePool(4)
    a, b = pool.take(2)
    pool.share([a])
    pool.share([a, b])
    assert pool.holders(a) == 3 and pool.holders(b) == 2 and pool.free_pages == 2 and pool.shared == 3
    pool.give_back([a, b])
    pool.give_back([a])
    assert pool.free_pages == 2 and pool.holders(a) == 1
    pool.give_back([b, a])
    assert pool.free_pages == 4 and pool.shared == 0
    for bad in ([a], [0], [5]):
        with pytest.raises(RuntimeError):
            pool.share(bad)
        with pytest.raises(RuntimeError):
            pool.give_back(bad)


def make_cache(max_tokens=64 * 40, window=None, state=True, slots=16):
    req = CacheRequest("window", 2, 4, window) if window else CacheRequest("full", 2, 4)
    return SequenceCache([(i, req, StateRequest((3,)) if state else None, None) for i in range(2)], max_tokens=max_tokens, max_slots=slots,
                         max_seq_len=4096, dtype=torch.float32, device="cpu")


class Mirror:
    """Writes tokens into a cache as a step would, and keeps what every slot must hold."""

    def __init__(self, cache):
        self.cache, self.rows, self.states, self.next = cache, {}, {}, 1.0

    def open(self):
        s = self.cache.open_slot()
        self.rows[s], self.states[s] = [], 0.0
        return s

    def write(self, slots, n):
        c = self.cache
        c.reserve([(s, c.length(s) + n) for s in slots])
        c.sync_tables()
        for s in slots:
            for i in range(c.length(s), c.length(s) + n):
                for g in c.groups:
                    page = int(g.table_dev[s, i // PAGE_TOKENS])
                    assert page == g.pages[s][i // PAGE_TOKENS] != 0 and g.pool.holders(page) == 1
                    g.k[:, page, :, i % PAGE_TOKENS] = self.next
                    g.v[:, page, :, i % PAGE_TOKENS] = -self.next
                self.rows[s].append(self.next)
                self.next += 1
            self.states[s] += self.next
            for t in c._state.values():
                t[s] = self.states[s]
            c.commit(s, c.length(s) + n)

    def check(self, first=0):
        c = self.cache
        held = {}
        for s, rows in self.rows.items():
            assert c.length(s) == len(rows)
            for g in c.groups:
                lo = g.first_live[s] * PAGE_TOKENS
                for i, v in enumerate(rows):
                    if i < lo:
                        continue
                    page = int(g.table_host[s, i // PAGE_TOKENS])
                    assert (g.k[:, page, :, i % PAGE_TOKENS] == v).all() and (g.v[:, page, :, i % PAGE_TOKENS] == -v).all()
                for p in g.pages[s]:
                    if p:
                        held[id(g), p] = held.get((id(g), p), 0) + 1
            for t in c._state.values():
                assert (t[s] == self.states[s]).all()
        for g in c.groups:
            for p in range(1, g.n_pages + 1):
                assert g.pool.holders(p) == held.get((id(g), p), 0)
            assert g.pool.free_pages == g.n_pages - len({p for i, p in held if i == id(g)})


@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("seed", range(6))
def test_forks_and_reordering_against_whole_copies(window, seed):
    """Random forks, reorderings, steps, rewinds and ends: every slot holds what it would with pages of its own."""
    rng = random.Random(seed)
    m = Mirror(make_cache(window=window, state=window is None or seed % 2 == 0))
    c = m.cache
    groups = []                                     # slots that belong together
    for _ in range(60):
        what = rng.random()
        if what < 0.25 and len(groups) < 4:
            s = m.open()
            m.write([s], rng.choice([1, 63, 64, 65, 130]))
            row = [s]
            for _ in range(rng.randrange(3)):
                f = c.fork(s)
                m.rows[f], m.states[f] = list(m.rows[s]), m.states[s]
                row.append(f)
            groups.append(row)
        elif what < 0.55 and groups:
            width = len(rng.choice(groups))
            rows = [r for r in groups if len(r) == width]
            parents = [[rng.randrange(width) for _ in r] for r in rows]
            was = {s: (list(m.rows[s]), m.states[s]) for r in rows for s in r}
            c.reorder(rows, parents)
            for r, up in zip(rows, parents):
                for s, p in zip(r, up):
                    m.rows[s], m.states[s] = list(was[r[p]][0]), was[r[p]][1]
        elif what < 0.9 and groups:
            chosen = [s for r in groups if rng.random() < 0.7 for s in r]
            if chosen and max(len(m.rows[s]) for s in chosen) < 500:
                try:
                    m.write(chosen, rng.choice([1, 1, 1, 2, 70]))
                except CacheFullError:
                    pass
        elif groups:
            row = groups.pop(rng.randrange(len(groups)))
            for s in row:
                c.close_slot(s)
                del m.rows[s], m.states[s]
        m.check()
    for row in groups:
        for s in row:
            c.close_slot(s)
    assert c.free_pages == c.n_pages


def test_a_full_pool_changes_nothing():
    c = make_cache(max_tokens=64 * 4)
    m = Mirror(c)
    s = m.open()
    m.write([s], 100)                               # two pages
    forks = [c.fork(s) for _ in range(4)]
    for f in forks:
        m.rows[f], m.states[f] = list(m.rows[s]), m.states[s]
    with pytest.raises(CacheFullError):             # four of the five want a page of their own, two are free
        c.reserve([(x, 101) for x in [s] + forks])
    m.check()
    m.write([forks[0], forks[1]], 1)
    m.check()
    with pytest.raises(CacheFullError):
        c.reserve([(forks[2], 101)])
    assert c.truncate(forks[2], 10) == 100 if c._state else True
    c.close_slot(forks[0])
    m.rows.pop(forks[0]), m.states.pop(forks[0])
    m.write([forks[2]], 1)
    m.check()


def test_pages_beyond_a_shared_length_are_not_shared_when_written():
    """A slot that reserved more than it kept hands its spare pages on with a reordering; each writer gets its own."""
    c = make_cache(state=False)
    m = Mirror(c)
    a = m.open()
    m.write([a], 64)
    b = c.fork(a)
    m.rows[b], m.states[b] = list(m.rows[a]), 0.0
    c.reserve([(a, 64 + 70)])                       # two spare pages
    c.reorder([[a, b]], [[0, 0]])
    m.write([a, b], 70)
    m.check()


def test_rewinding_to_the_own_length_gives_spare_pages_back():
    """What was reserved and not kept goes back, to the pool or to its other holders, and the slot goes on as before."""
    for window, state in ((None, False), (None, True), (100, False)):
        c = make_cache(window=window, state=state)
        m = Mirror(c)
        a = m.open()
        m.write([a], 130)
        m.check()
        free = c.free_pages
        c.reserve([(a, 130 + 200)])
        assert c.free_pages < free
        b = c.fork(a)
        m.rows[b], m.states[b] = list(m.rows[a]), m.states[a]
        for s in (a, b):
            assert c.truncate(s, 130) == 130 == c.length(s)
        assert c.free_pages == free
        m.check()
        m.write([a, b], 70)
        m.check()
        assert c.truncate(a, 10 ** 6) == 200


def test_reordering_refuses_what_is_no_permutation_of_open_slots():
    c = make_cache()
    a, b = c.open_slot(), c.open_slot()
    for slots, parents in (([[a, a]], [[0, 1]]), ([[a, b]], [[0, 2]]), ([[a, b]], [[0, -1]]), ([[a, b]], [[0]]), ([[a], [b, 7]], [[0], [0, 1]])):
        with pytest.raises(ValueError):
            c.reorder(slots, parents)
    with pytest.raises(RuntimeError):
        c.reorder([[a, 9]], [[0, 1]])
    with pytest.raises(RuntimeError):
        c.fork(11)


def test_tree_facts():
    rng = random.Random(0)
    for n in (1, 31, 32, 33, 64, 100, 256):
        parents = random_tree(rng, n, 0.5)
        masks, depths = tree_facts(parents, (n + 31) // 32 + 1)
        bits = np.unpackbits(masks.view(np.uint8), axis=1, bitorder="little")[:, :n].astype(bool)
        assert (bits == ancestors(parents)).all() and masks.shape == (n, (n + 31) // 32 + 1)
        assert (depths == bits.sum(axis=1) - 1).all()


def test_prompt_lookup_drafts_what_followed_before():
    draft = PromptLookup(longest=2, branches=2, length=3)
    tokens, parents = draft([1, 2, 3, 4, 9, 1, 2, 3, 5, 8, 1, 2], 10)
    # the latest place first (3 5 8), then 3 4 9 shares its first token
    assert tokens == [3, 5, 8, 4, 9] and parents == [-1, 0, 1, 0, 3]
    assert draft([1, 2, 3, 4, 9, 1, 2, 3, 5, 8, 1, 2], 2) == ([3, 5], [-1, 0])
    assert draft([1, 2, 3], 5) == ([], []) and draft([7], 5) == ([], [])
    for n in range(1, 40):
        seq = [random.Random(n).randrange(3) for _ in range(n)]
        tokens, parents = draft(seq, 6)
        assert len(tokens) == len(parents) <= 6 and all(-1 <= p < i for i, p in enumerate(parents))
        assert len({(p, t) for p, t in zip(parents, tokens)}) == len(tokens)


class _Cache:
    max_seq_len = 100

    def length(self, slot):
        return 10


def test_beam_decisions():
    """Stop tokens end a beam if they are among the best, missing candidates leave empty beams, a search ends when nothing better goes on."""
    b = object.__new__(BeamSearch)
    b.beams, b.stop, b.penalty = 2, frozenset([7]), 1.0
    s = _Search([0, 1], [[]], [0.0])
    assert b._advance(s, [-1.0, -2.0, -3.0, -4.0], [0, 0, 0, 0], [5, 7, 6, 8], 9, _Cache())
    assert s.tokens == [[5], [6]] and s.scores == [-1.0, -3.0] and s.next_parents == [0, 0]
    assert [(r.tokens, r.log_prob, r.score, r.finish_reason) for r in s.done] == [([], -2.0, -2.0, "stop")]
    # an ending that is not among the best two is passed over
    assert b._advance(s, [-1.5, -2.5, -2.6, -9.0], [0, 0, 0, 1], [4, 3, 7, 2], 9, _Cache())
    assert s.tokens == [[5, 4], [5, 3]] and s.next_parents == [0, 0] and len(s.done) == 1
    # one candidate only: the other beam stands empty
    assert b._advance(s, [-1.6, float("-inf"), float("-inf"), float("-inf")], [1, -1, -1, -1], [2, -1, -1, -1], 9, _Cache())
    assert s.tokens == [[5, 3, 2], [5, 3, 2]] and s.scores == [-1.6, float("-inf")] and s.next_parents == [1, 1]
    # two ended, none that goes on is more probable
    assert not b._advance(s, [-1.7, -2.8, -5.0, -6.0], [0, 0, 0, 0], [7, 1, 2, 3], 9, _Cache())
    assert len(s.done) == 2
    t = _Search([0, 1], [[]], [0.0])
    assert not b._advance(t, [-1.0, -2.0], [0, 0], [1, 2], 1, _Cache())
    assert [(r.tokens, r.finish_reason) for r in t.done] == [([1], "length"), ([2], "length")]


def test_refusals_without_a_gpu():
    cpu = torch.zeros(4, 8)
    ints = torch.zeros((1, 4), dtype=torch.int32)
    with pytest.raises(KernelError):
        ops.beam_select(cpu, torch.zeros(1, 4), 2)
    with pytest.raises(KernelError):
        ops.reorder_states([cpu], ints, ints)
    with pytest.raises(KernelError):
        ops.copy_pages([torch.zeros(1, 2, 1, 64, 4)], ints[0], ints[0])
    with pytest.raises(KernelError):
        ops.tree_commit(ints[0], ints[0], ints[0], torch.zeros(2, dtype=torch.int32), ints[0, :1], ints[0, :1], 1, 4, [], ints)
    with pytest.raises(KernelError):
        ops.attention_tree(cpu, torch.zeros(2, 1, 64, 8), torch.zeros(2, 1, 64, 8), ints, torch.zeros(2, dtype=torch.int32), ints[0, :1], ints[0, :1],
                           torch.zeros((4, 1), dtype=torch.int32), 1, 4, 4, 1, 1, 8, 1.0, cpu)
    for beams in (0, 33):
        with pytest.raises(ValueError):
            BeamSearch(None, beams)

    class Engine:
        def takes_trees(self):
            return False
    with pytest.raises(ValueError):
        DraftedLoop(Engine(), PromptLookup())
    for nodes in (0, 257):
        with pytest.raises(ValueError):
            DraftedLoop(Engine(), PromptLookup(), max_nodes=nodes)


def test_command_line_options():
    o = cli.parse_opts(["m", "--beams", "4", "--draft", "16"])
    assert (o.beams, o.draft) == (4, 16)
    for args in (["--beams", "4", "--draft", "16"], ["--beams", "-1"], ["--draft", "-2"]):
        with pytest.raises(cli.UsageError):
            cli.cmd_run(cli.parse_opts(["m", "-p", "1"] + args))
    assert plain_walk([], [], []) == ([], -1)


def test_a_search_that_finds_nothing_prints_an_empty_line(monkeypatch, capsys):
    """Logits that are no numbers leave a beam search without results."""
    class Llm:
        last_stats = None

        def beam_search(self, prompts, **kw):
            return [[] for _ in prompts]
    monkeypatch.setattr(cli, "_llm", lambda *a, **k: Llm())
    cli.cmd_run(cli.parse_opts(["m", "-p", "1,2;3", "--beams", "2"]))
    assert capsys.readouterr().out.split("\n")[:2] == ["", ""]


def test_drafted_batches_are_no_larger_than_a_launch_takes():
    class Slots:
        free_slots = 5000

    class Cache:
        max_seq_len, free_pages, slots = 100, 5000, Slots()

    class Engine:
        cache = Cache()

        def takes_trees(self):
            return True
    loop = DraftedLoop(Engine(), PromptLookup(), batch_size=3000)
    taken = []
    loop._run_batch = lambda prompts, results, ids, max_new: taken.append(len(ids))
    loop.run([[1]] * 2500, 4)
    assert taken == [1024, 1024, 452]
