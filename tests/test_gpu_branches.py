"""The operators that hold several continuations of a sequence, each alone against its plain statement in 64 bits."""
import itertools
import math
import random

import numpy as np
import pytest
import torch

from ghost_infer_b200.kernels import ops
from ghost_infer_b200.kernels.library import KernelError
from branch_cases import ancestors, mask_words, plain_beam_select, plain_tree_attention, plain_walk, random_tree

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def randn(*shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ---- beam search's choice -------------------------------------------------------------------------------------------------
def check_beams(logits, scores, width):
    got = ops.beam_select(logits, scores, width)
    want = plain_beam_select(logits.cpu().double().numpy(), scores.cpu().double().numpy(), width)
    assert [t.dtype for t in got] == [F32, torch.int32, torch.int32] and all(tuple(t.shape) == want[0].shape for t in got)
    assert (got[1].cpu().numpy() == want[1]).all() and (got[2].cpu().numpy() == want[2]).all()
    value = got[0].cpu().double().numpy()
    live = np.isfinite(want[0])
    assert (value[~live] == -np.inf).all()
    value, exact = value[live], want[0][live]
    # the log sum carries the 32-bit sums' errors: 64 additions and an exponential good to 2^-22 a number, below 1e-5; the result
    # is rounded to 32 bits
    assert (np.abs(value - exact) <= 1e-5 + 2.0 ** -24 * np.abs(exact)).all()


@pytest.mark.parametrize("seqs,beams,vocab,width", [(1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 5, 4), (1, 4, 128256, 8), (3, 2, 4096, 64), (2, 16, 16385, 32),
                                                     (1, 64, 300, 64), (5, 5, 32003, 10), (300, 1, 1000, 3), (1, 1, 50001, 64)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_beam_select(seqs, beams, vocab, width, dtype):
    logits = randn(seqs * beams, vocab, dtype=dtype, seed=vocab + width, scale=3.0)
    check_beams(logits, randn(seqs, beams, seed=1, scale=4.0), width)


@pytest.mark.parametrize("shift", range(8))
def test_beam_select_rows_that_start_anywhere(shift):
    """Views whose rows start on no boundary and lie further apart than they are long."""
    for dtype, vocab in ((BF16, 5003), (F32, 4099), (BF16, 9), (F32, 3)):
        whole = randn(6, vocab + 13, dtype=dtype, seed=shift, scale=2.0)
        check_beams(whole[:, shift:shift + vocab], randn(2, 3, seed=shift), min(11, 3 * vocab))


def test_beam_select_ties_go_to_the_lowest_place():
    equal = torch.full((6, 40000), 0.5, device=DEV)
    check_beams(equal, torch.zeros(2, 3, device=DEV), 40)
    few = torch.zeros((4, 3000), dtype=BF16, device=DEV)
    few[:, 100::100] = 1.0
    check_beams(few, torch.zeros(1, 4, device=DEV), 64)
    # the first step of a search: every beam is the same one
    row = randn(1, 128256, seed=3, scale=3.0)
    check_beams(row.expand(8, -1).contiguous(), torch.zeros(2, 4, device=DEV), 8)
    signs = torch.zeros((2, 64), device=DEV)
    signs[:, ::2] = -0.0
    check_beams(signs, torch.zeros(1, 2, device=DEV), 10)


def test_beam_select_infinities_and_what_is_no_number():
    inf, nan = float("inf"), float("nan")
    logits = randn(8, 20011, seed=5, scale=2.0)
    logits[0, :] = -inf                          # a beam whose mask left nothing
    logits[1, 7] = inf
    logits[2, ::2] = nan
    logits[3, 1:] = -inf                         # one token left
    logits[4, :] = torch.finfo(F32).min          # masked by the type's lowest value throughout
    logits[5, 5:] = torch.finfo(F32).min
    scores = torch.zeros(2, 4, device=DEV)
    scores[1, 2] = -inf                          # a beam that does not exist
    check_beams(logits, scores, 16)
    scores[1, 3] = nan
    check_beams(logits, scores, 64)
    check_beams(torch.full((4, 9000), -inf, device=DEV), torch.zeros(2, 2, device=DEV), 5)
    few = torch.full((4, 9000), -inf, device=DEV)
    few[1, 8999], few[2, 0], few[3, 4500] = 1.0, 2.0, -3.0
    check_beams(few, torch.tensor([[0.0, -1.0], [-2.0, 0.25]], device=DEV), 4)


def test_beam_select_graph_and_stream():
    logits, scores = randn(8, 32003, seed=8, scale=3.0), randn(2, 4, seed=9)
    want = [t.clone() for t in ops.beam_select(logits, scores, 8)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.beam_select(logits, scores, 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.beam_select(logits, scores, 8)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, other))
    logits.copy_(randn(8, 32003, seed=10, scale=3.0))
    graph.replay()
    assert torch.equal(got[2], ops.beam_select(logits, scores, 8)[2])


def check_beams_closely(logits, scores, width, off):
    """`off`: what the log sum may be off by; added to a large logit in 64 bits it may become the number next to the plain one's."""
    got = [t.cpu().numpy() for t in ops.beam_select(logits, scores, width)]
    want = plain_beam_select(logits.cpu().double().numpy(), scores.cpu().double().numpy(), width)
    assert (got[1] == want[1]).all() and (got[2] == want[2]).all()
    assert (np.abs(got[0].astype(np.float64) - want[0]) <= off + 2.0 ** -52 * float(logits.abs().max()) + 2.0 ** -24 * np.abs(want[0])).all()


@pytest.mark.parametrize("shift", [-1e6, -1e4, -1e3, -100.0, 0.0, 100.0, 1e3, 1e4, 1e6])
def test_beam_select_log_sums_of_rows_far_from_zero(shift):
    """The error of a log sum does not grow with the logits.  A number's exponent is rounded twice and scaled by a 32-bit log2(e)
    (2^-22.8 of it in all), under a row's probabilities at most ln 40,000 = 10.6 of it; an exponential is good to 2^-22, 15 additions lie
    on a number's way: below 2.6e-6."""
    logits = randn(4, 40000, seed=int(abs(shift)), scale=3.0) + shift
    # (two beams' candidates may lie nearer to each other than that: one beam a sequence)
    check_beams_closely(logits, randn(4, 1, seed=2), 16, 2.6e-6)


@pytest.mark.parametrize("top", [20.0, 50.0, 120.0, 1020.0, 10020.0, -3e5])
def test_beam_select_sure_tokens(top):
    """Next to a token that has all of the probability the others' sum is nothing: no error but the result's own rounding, and no
    log probability above zero."""
    logits = randn(3, 20000, seed=4) - 200.0 + top
    logits[:, 777] = top
    scores = torch.zeros(3, 1, device=DEV)
    check_beams_closely(logits, scores, 5, 1e-7)
    assert (ops.beam_select(logits, scores, 1)[0] == 0).all()


@pytest.mark.parametrize("value", [-4e9, -6e9, -1e9, -1e11, -1e12, -1e15, -1e25, -1e30, 1e9, 1e25])
def test_beam_select_rows_of_one_finite_value(value):
    """A row that a mask filled throughout with a large finite number still has tokens, each as likely as another."""
    check_beams_closely(torch.full((2, 9000), value, device=DEV), torch.tensor([[-1.0], [0.5]], device=DEV), 6, 2.6e-6)
    mixed = torch.full((2, 9000), value, device=DEV)
    mixed[0, 4000:4003] = abs(value)
    check_beams_closely(mixed, torch.tensor([[-1.0], [0.5]], device=DEV), 6, 2.6e-6)


@pytest.mark.parametrize("dtype,seqs,beams,vocab", [(F32, 1, 8, 32003), (F32, 1, 2, 32003), (F32, 8, 8, 128256), (F32, 20, 5, 70001), (BF16, 2, 8, 32003), (BF16, 30, 4, 50257)])
def test_beam_select_equal_beams_tie_wherever_their_rows_lie(dtype, seqs, beams, vocab):
    """Rows that start on different boundaries, and are cut at different places by the calls' many blocks, have the same sum."""
    row = randn(1, vocab, dtype=dtype, seed=vocab + beams, scale=3.0)
    logits = row.expand(seqs * beams, -1).contiguous()
    got = ops.beam_select(logits, torch.full((seqs, beams), -2.5, device=DEV), beams)
    best = torch.arange(vocab, device=DEV)[row[0] == row[0].max()].tolist()
    want = [(j, t) for j in range(beams) for t in best][:beams]
    assert got[1].tolist() == [[j for j, _ in want]] * seqs and got[2].tolist() == [[t for _, t in want]] * seqs
    assert (got[0] == got[0][0, 0]).all()


def test_beam_select_does_not_depend_on_the_rest_of_the_call():
    logits, scores = randn(80, 65000, seed=6, scale=3.0), randn(20, 4, seed=7)
    together = ops.beam_select(logits, scores, 12)
    for s in (0, 7, 19):
        alone = ops.beam_select(logits[4 * s:4 * s + 4], scores[s:s + 1].contiguous(), 12)
        assert all(torch.equal(a[s:s + 1], b) for a, b in zip(together, alone))
    for dtype, vocab in ((F32, 65003), (BF16, 65003)):
        rows = randn(4, vocab, dtype=dtype, seed=8, scale=3.0)
        want = ops.beam_select(rows, scores[:1].contiguous(), 20)
        for shift in range(1, 9):
            wide = torch.full((4, vocab + 16 + shift), 60.0, dtype=dtype, device=DEV)      # (what lies around a row is larger than all of it)
            wide[:, shift:shift + vocab] = rows
            got = ops.beam_select(wide[:, shift:shift + vocab], scores[:1].contiguous(), 20)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- states and pages -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("beams", [1, 2, 4, 5, 8, 9, 16, 17, 40, 41, 64])
@pytest.mark.parametrize("kind", ["float", "mixed"])
def test_reorder_states(beams, kind):
    rng = random.Random(beams)
    seqs = 3
    rows = seqs * beams + 2
    if kind == "float":
        states = [randn(rows, 16, 66, seed=i) for i in range(3)] + [randn(rows, 4100, seed=7)]
    else:
        states = [randn(rows, 37, dtype=BF16, seed=1), randn(rows, 5, seed=2), torch.arange(rows * 3, device=DEV, dtype=torch.uint8).view(rows, 3),
                  randn(rows, 8, dtype=BF16, seed=3), randn(rows, 2, 3, seed=4).double()]
    order = list(range(rows))
    rng.shuffle(order)
    slots = [order[s * beams:(s + 1) * beams] for s in range(seqs)]
    parents = [[rng.randrange(beams) for _ in range(beams)], list(range(beams - 1, -1, -1)), [rng.choice([j, 0]) for j in range(beams)]]
    parents[2][beams // 2] = -1                       # nobody: stays
    parents[1][0] = beams                             # no beam of this sequence: stays
    if beams > 2:
        slots[0][1] = -1                              # a padding row: nothing is moved to it or from it
    want = [t.clone() for t in states]
    for t, w in zip(states, want):
        for row, up in zip(slots, parents):
            for j, p in enumerate(up):
                if row[j] >= 0 and 0 <= p < beams and row[p] >= 0:
                    w[row[j]] = t[row[p]]
    ops.reorder_states(states, i32(slots), i32(parents))
    for t, w in zip(states, want):
        assert torch.equal(t, w)


def test_reorder_states_many_tensors_and_large_rows():
    states = [randn(5, 1000 + i, seed=i) for i in range(67)] + [randn(5, 300_001, seed=99)]
    want = [t[[2, 1, 2, 0, 4]].clone() for t in states]
    ops.reorder_states(states, i32([[0, 1, 2, 3]]), i32([[2, 1, 2, 0]]))
    assert all(torch.equal(t, w) for t, w in zip(states, want))
    ops.reorder_states([], i32([[0, 1]]), i32([[1, 0]]))
    ops.reorder_states([torch.zeros(4, 0, device=DEV)], i32([[0, 1]]), i32([[1, 0]]))


@pytest.mark.parametrize("dtype,dims", [(BF16, (64, 64)), (F32, (16, 24)), (BF16, (5, 40)), (BF16, (6, 6))])
def test_copy_pages(dtype, dims):
    pages = [randn(3, 12, 2, 64, dims[0], dtype=dtype, seed=1), randn(3, 12, 2, 64, dims[1], dtype=dtype, seed=2)]
    want = [t.clone() for t in pages]
    src, dst, rows = [4, 4, 9, 11, 0], [1, 2, 3, 5, 6], [1, 64, 33, 0, 77]
    for t in want:
        for a, b, n in zip(src, dst, rows):
            t[:, b, :, :n] = t[:, a, :, :n]
    ops.copy_pages(pages, i32(src), i32(dst), i32(rows))
    assert all(torch.equal(a, b) for a, b in zip(pages, want))
    ops.copy_pages(pages, i32([7, 12, -1, 8]), i32([10, 3, 4, 99]))          # pages that are not there are passed over
    for t in want:
        t[:, 10] = t[:, 7]
    assert all(torch.equal(a, b) for a, b in zip(pages, want))
    ops.copy_pages(pages, i32([]), i32([]))


# ---- the walk through a tree ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F32, 16), (BF16, 5), (BF16, 6)])
@pytest.mark.parametrize("sizes,pos0", [([1], [0]), ([26], [50]), ([7, 0, 64, 1, 33], [63, 5, 130, 64, 0]), ([256, 200], [40, 191]), ([40] * 9, list(range(30, 120, 10)))])
def test_tree_commit(dtype, dim, sizes, pos0):
    rng = random.Random(sum(sizes) + dim)
    layers, kv = 2, 3
    trees = [random_tree(rng, n, 0.6) for n in sizes]
    tokens = [[rng.randrange(3) for _ in t] for t in trees]                 # few tokens: siblings that are alike
    picks = [[rng.randrange(3) for _ in t] for t in trees]
    per = [(p + n + 63) // 64 for p, n in zip(pos0, sizes)]
    max_pages = max(per) + 1
    total = sum(per) + 1
    order = list(range(1, total))
    rng.shuffle(order)
    slots = list(range(len(sizes)))
    rng.shuffle(slots)
    table = [[0] * max_pages for _ in sizes]
    for b, s in enumerate(slots):
        for i in range(per[b]):
            table[s][i] = order.pop()
    pages = [randn(layers, total, kv, 64, dim, dtype=dtype, seed=1), randn(layers, total, kv, 64, 2 * dim, dtype=dtype, seed=2)]
    want = [t.clone() for t in pages]
    max_nodes = max(sizes)
    want_path, want_next = [], []
    for b, s in enumerate(slots):
        path, nxt = plain_walk(picks[b], tokens[b], trees[b])
        want_path.append(path + [-1] * (max_nodes - len(path)))
        want_next.append(nxt)
        for t, w in zip(pages, want):
            for i, node in enumerate(path):
                a, c = pos0[b] + node, pos0[b] + i
                w[:, table[s][c // 64], :, c % 64] = t[:, table[s][a // 64], :, a % 64]
    flat = lambda rows: i32([x for row in rows for x in row])
    cu = i32([0] + list(itertools.accumulate(sizes)))
    args = (flat(picks), flat(tokens), flat(trees), cu, i32(slots), i32(pos0), len(sizes), max_nodes)
    path, counts, nexts = ops.tree_commit(*args, pages, i32(table))
    assert path.cpu().tolist() == want_path and nexts.cpu().tolist() == want_next
    assert counts.cpu().tolist() == [sum(x >= 0 for x in row) for row in want_path]
    assert all(torch.equal(a, b) for a, b in zip(pages, want))
    again = ops.tree_commit(*args, [], i32(table))                            # the walk alone
    assert all(torch.equal(a, b) for a, b in zip((path, counts, nexts), again))


def test_tree_commit_parents_that_are_no_tree():
    """A parent that does not come before its node is nobody's parent: the walk still ends, and stays inside."""
    parents, tokens = [0, 2, 5, 1, -7, 99, 3], [1] * 7
    path, counts, nexts = ops.tree_commit(i32([1] * 7), i32(tokens), i32(parents), i32([0, 7]), i32([-1]), i32([0]), 1, 8, [], i32([[0]]))
    want, nxt = plain_walk([1] * 7, tokens, parents)
    assert path[0].cpu().tolist() == want + [-1] * (8 - len(want)) and nexts.tolist() == [nxt]


def test_tree_commit_padding_and_rows_outside():
    """A slot of -1 and positions past the table move nothing."""
    pages = [randn(1, 3, 1, 64, 8, seed=1)]
    want = pages[0].clone()
    args = lambda slot, pos: (i32([5, 5, 5]), i32([0, 4, 5]), i32([-1, 0, 0]), i32([0, 3]), i32([slot]), i32([pos]), 1, 3, pages, i32([[1]]))
    for slot, pos in ((-1, 0), (0, 64), (0, 6400)):
        path, counts, nexts = ops.tree_commit(*args(slot, pos))
        assert path.cpu().tolist() == [[0, 2, -1]] and counts.tolist() == [2] and nexts.tolist() == [5]
        assert torch.equal(pages[0], want)


# ---- attention over a tree --------------------------------------------------------------------------------------------------
class TreeCase:
    """Paged keys and values of several sequences with their trees; everything that no node may look at holds NaN."""

    def __init__(self, sizes, pos0, heads, kv, dim, dtype, seed=0, seen=None, extra_cols=0, scale=1.0):
        rng = random.Random(seed)
        self.sizes, self.pos0, self.heads, self.kv, self.dim, self.dtype = sizes, pos0, heads, kv, dim, dtype
        per = [(p + n + 63) // 64 for p, n in zip(pos0, sizes)]
        total = sum(per) + 3
        order = list(range(1, total))
        rng.shuffle(order)
        self.slots = list(range(len(sizes)))
        rng.shuffle(self.slots)
        self.table = [[total - 1] * (max(per) + 1) for _ in sizes]
        k, v = (torch.full((total, kv, 64, dim), float("nan"), dtype=dtype) for _ in range(2))
        k[0] = v[0] = 0
        g = torch.Generator().manual_seed(seed)
        self.dense = []
        for b, s in enumerate(self.slots):
            n = pos0[b] + sizes[b]
            kd, vd = (torch.randn(n, kv, dim, generator=g).to(dtype) for _ in range(2))
            self.dense.append((kd, vd))
            for i in range(per[b]):
                page = order.pop()
                self.table[s][i] = page
                rows = min(64, n - 64 * i)
                k[page, :, :rows] = kd[64 * i:64 * i + rows].transpose(0, 1)
                v[page, :, :rows] = vd[64 * i:64 * i + rows].transpose(0, 1)
        self.k, self.v = k.to(DEV), v.to(DEV)
        self.q = (torch.randn(sum(sizes), heads * dim + extra_cols, generator=g) * scale).to(dtype).to(DEV)
        self.seen = seen or [ancestors(random_tree(rng, n)) for n in sizes]
        self.words = max(1, (max(sizes) + 31) // 32)
        self.masks = mask_words(self.seen, self.words).to(DEV)
        self.cu, self.table_dev, self.slots_dev, self.pos0_dev = (i32(x) for x in ([0] + list(itertools.accumulate(sizes)), self.table, self.slots, pos0))

    def run(self, **kw):
        out = torch.full((sum(self.sizes), self.heads * self.dim), 7.0, dtype=self.dtype, device=DEV)
        longest = max(p + n for p, n in zip(self.pos0, self.sizes))
        a = dict(q=self.q, kcache=self.k, vcache=self.v, block_table=self.table_dev, cu_seqlens=self.cu, seq_slots=self.slots_dev, seq_pos0=self.pos0_dev,
                 masks=self.masks, n_seqs=len(self.sizes), max_nodes=max(self.sizes), max_kv_len=longest, n_heads=self.heads, n_kv=self.kv, head_dim=self.dim,
                 scale=self.dim ** -0.5, out=out)
        a.update(kw)
        return ops.attention_tree(**a)

    def check(self, got, only=None):
        got = got.float().cpu().double().numpy().reshape(-1, self.heads, self.dim)
        at = 0
        for b, n in enumerate(self.sizes):
            if only is None or b in only:
                kd, vd = (t.double().numpy() for t in self.dense[b])
                q = self.q[at:at + n, :self.heads * self.dim].cpu().double().numpy().reshape(n, self.heads, self.dim)
                seen = np.concatenate([np.ones((n, self.pos0[b]), dtype=bool), self.seen[b]], axis=1)
                want, spread, most = plain_tree_attention(q, kd, vd, seen, self.dim ** -0.5)
                # A score is off by at most (dim + 2) roundings of its products' sum (2^-23 each on tensor cores, which may
                # truncate), which moves a weight by that much relatively, numerator and denominator; the sums over the keys
                # are off by their length in roundings; exponentials by 2^-21.  In 16 bits a weight is rounded (2^-8), and the result.
                keys = self.pos0[b] + n
                weight = 2 * (self.dim + 2) * 2.0 ** -23 * most + 2 * keys * 2.0 ** -23 + 2.0 ** -20
                if self.dtype == BF16:
                    bound = (weight + 2.0 ** -8) * spread * (1 + 2.0 ** -7) + 2.0 ** -8 * np.abs(want) + 1e-30
                else:
                    bound = weight * spread + 2.0 ** -23 * np.abs(want) + 1e-30
                err = np.abs(got[at:at + n] - want)
                assert np.isfinite(got[at:at + n]).all(), f"sequence {b}: not finite"
                assert (err <= bound).all(), f"sequence {b}: {float((err / bound).max()):.2f} times what the arithmetic allows"
            at += n


SHAPES = [(4, 4, 64), (4, 2, 128), (6, 2, 64), (32, 8, 128), (3, 1, 128), (5, 1, 48), (2, 1, 256), (7, 7, 20), (8, 1, 33), (16, 1, 128)]


@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_shapes(heads, kv, dim, dtype):
    c = TreeCase([5, 1, 17], [70, 0, 200], heads, kv, dim, dtype, seed=dim)
    c.check(c.run())


@pytest.mark.parametrize("sizes,pos0", [([1], [0]), ([1], [1]), ([1], [63]), ([1], [64]), ([1], [4000]), ([64], [0]), ([65], [63]), ([256], [10]), ([31, 32, 33], [1, 64, 127]),
                                        ([26], [1500]), ([100, 3, 1, 60], [700, 5000, 64, 0]), ([2] * 40, list(range(0, 800, 20)))])
@pytest.mark.parametrize("dtype,heads,kv,dim", [(F32, 4, 2, 64), (BF16, 4, 2, 64), (BF16, 8, 2, 128), (BF16, 3, 1, 128), (BF16, 4, 4, 128), (BF16, 2, 1, 80)])
def test_tree_attention_lengths(sizes, pos0, dtype, heads, kv, dim):
    c = TreeCase(sizes, pos0, heads, kv, dim, dtype, seed=sum(sizes), scale=2.0)
    c.check(c.run())


@pytest.mark.parametrize("dtype,dim", [(F32, 64), (BF16, 64), (BF16, 128), (BF16, 96)])
def test_tree_attention_masks(dtype, dim):
    """Any mask, nodes that see nothing (zeros), mask words past the tree, nodes that see all of it."""
    rng = np.random.default_rng(dim)
    sizes, pos0 = [40, 33, 70, 5], [0, 100, 0, 64]
    seen = [rng.random((n, n)) < 0.3 for n in sizes]
    seen[0][3] = False
    seen[0][20] = False
    seen[2][:] = True
    seen[3][:] = False
    c = TreeCase(sizes, pos0, 4, 2, dim, dtype, seed=3, seen=seen)
    c.masks[:40, 1] |= -(1 << 8)              # bits of nodes that the first tree does not have
    got = c.run()
    c.check(got)
    assert (got[3] == 0).all() and (got[20] == 0).all()
    # wider mask rows than needed
    wide = torch.full((c.masks.shape[0], c.words + 3), -1, dtype=torch.int32, device=DEV)
    wide[:, :c.words] = c.masks
    assert torch.equal(c.run(masks=wide), got)


@pytest.mark.parametrize("dtype,dim", [(F32, 64), (BF16, 64), (BF16, 128), (BF16, 40)])
def test_tree_attention_values_that_are_no_numbers(dtype, dim):
    """A node whose key or value is no number (or infinite) spoils those that see it and nobody else."""
    rng = random.Random(1)
    trees = [random_tree(rng, 20, 0.2), random_tree(rng, 50, 0.3)]
    seen = [ancestors(t) for t in trees]
    c = TreeCase([20, 50], [50, 10], 4, 2, dim, dtype, seed=5, seen=seen)
    clean = c.run()
    bad = {0: [7, 19], 1: [30]}
    for b, nodes in bad.items():
        for node in nodes:
            at = c.pos0[b] + node
            page = c.table[c.slots[b]][at // 64]
            c.v[page, :, at % 64, node % dim] = float("nan")
            c.v[page, 0, at % 64, 3] = float("inf")
            c.k[page, :, at % 64, 1] = float("nan")
    got = c.run()
    at = 0
    for b, n in enumerate(c.sizes):
        for i in range(n):
            if any(seen[b][i, node] for node in bad[b]):
                assert not torch.isfinite(got[at + i].float()).all()
            else:
                assert torch.equal(got[at + i], clean[at + i]), (b, i)
        at += n


@pytest.mark.parametrize("dtype,dim", [(F32, 64), (BF16, 128), (BF16, 72)])
def test_tree_attention_rows_strides_and_padding(dtype, dim):
    """Packed rows, output rows inside a wider tensor, padding sequences, too small a length given: the rows around stay."""
    c = TreeCase([9, 30], [130, 77], 4, 2, dim, dtype, seed=8, extra_cols=4 * dim)
    want = c.run()
    c.check(want)
    wide = torch.full((39, 4 * dim + 16), 5.0, dtype=dtype, device=DEV)
    c.run(out=wide[:, 8:8 + 4 * dim])
    assert torch.equal(wide[:, 8:8 + 4 * dim], want) and (wide[:, :8] == 5).all() and (wide[:, 8 + 4 * dim:] == 5).all()
    # rows behind the last sequence are left as they were; a padding sequence (slot -1) reads the trash page
    more = torch.cat([c.q, c.q[:3]])
    out = torch.full((42, 4 * dim), 3.0, dtype=dtype, device=DEV)
    masks = torch.cat([c.masks, c.masks[:3]])
    c.run(q=more, out=out, masks=masks)
    assert torch.equal(out[:39], want) and (out[39:] == 3).all()
    padded = torch.full((42, 4 * dim), 3.0, dtype=dtype, device=DEV)
    c.run(q=more, out=padded, masks=masks, cu_seqlens=i32([0, 9, 39, 40]), seq_slots=i32(c.slots + [-1]), seq_pos0=i32(c.pos0 + [0]), n_seqs=3)
    assert torch.equal(padded[:39], want) and torch.isfinite(padded[39].float()).all() and (padded[40:] == 3).all()
    c.check(c.run(max_kv_len=1))
    c.check(c.run(max_kv_len=100000))


@pytest.mark.parametrize("dtype,dim,shift", [(BF16, 128, 1), (BF16, 64, 4), (F32, 64, 1), (BF16, 128, 8)])
def test_tree_attention_rows_on_any_boundary(dtype, dim, shift):
    """Queries and output that start on no 16-byte boundary, rows whose distance is no multiple of one."""
    c = TreeCase([9, 40], [130, 77], 4, 2, dim, dtype, seed=9)
    want = c.run()
    q = torch.zeros((49, 4 * dim + shift), dtype=dtype, device=DEV)
    q[:, shift:] = c.q
    wide = torch.zeros((49, 4 * dim + 2 * shift), dtype=dtype, device=DEV)
    c.check(c.run(q=q[:, shift:]))
    c.check(c.run(out=wide[:, shift:shift + 4 * dim]))
    c.check(c.run(q=q[:, shift:], out=wide[:, shift:shift + 4 * dim]))
    assert (wide[:, :shift] == 0).all() and (wide[:, shift + 4 * dim:] == 0).all()
    c.check(want)


@pytest.mark.parametrize("dtype,dim", [(F32, 64), (BF16, 128), (BF16, 72)])
def test_tree_attention_slots_and_lengths_that_are_not_there(dtype, dim):
    """A slot past the table's last row reads the trash page, as -1 does; offsets past the rows leave the rest out."""
    c = TreeCase([9, 30], [130, 77], 4, 2, dim, dtype, seed=8)
    want = c.run()
    c.k[0], c.v[0] = 0.5, 0.25
    for slot in (2, 1 << 20, -1, -(1 << 30)):
        got = c.run(seq_slots=i32([c.slots[0], slot]))
        # (107 keys at most: the sums of weights and of values, a weight's and the result's rounding to 16 bits)
        off = 0.25 * (2 * 107 * 2.0 ** -24 + (2.0 ** -7 + 2.0 ** -15 if dtype == BF16 else 2.0 ** -23))
        assert torch.equal(got[:9], want[:9]) and ((got[9:].float() - 0.25).abs() <= off).all()
    wide = torch.full((60, 4 * dim), 3.0, dtype=dtype, device=DEV)
    got = c.run(cu_seqlens=i32([0, 9, 50]), max_nodes=50, out=wide[:39], masks=torch.cat([c.masks, torch.zeros_like(c.masks)], dim=1))
    assert torch.equal(got[:9], want[:9]) and (wide[39:] == 3).all()
    c.check(c.run(cu_seqlens=i32([0, 9, 2000]), max_nodes=30, seq_pos0=c.pos0_dev))
    for cu in ([-5, 0, 0], [50, 60, 70], [0, 0, -3]):
        assert (c.run(cu_seqlens=i32(cu)) == 7).all()


def test_tree_commit_slots_and_lengths_that_are_not_there():
    pages = [randn(1, 3, 1, 64, 8, seed=1)]
    want = pages[0].clone()
    for slot in (1, 1 << 20):
        path, counts, nexts = ops.tree_commit(i32([5, 5, 5]), i32([0, 4, 5]), i32([-1, 0, 0]), i32([0, 3]), i32([slot]), i32([0]), 1, 3, pages, i32([[1]]))
        assert path.tolist() == [[0, 2, -1]] and torch.equal(pages[0], want)
    for cu in ([0, 200], [-4, 3], [7, 9]):
        path, counts, nexts = ops.tree_commit(i32([5, 5, 5]), i32([0, 4, 6]), i32([-1, 0, 0]), i32(cu), i32([0]), i32([0]), 1, 8, pages, i32([[1]]))
        n = 1 if cu[0] == 0 else 0
        assert counts.tolist() == [n] and path[0].tolist() == [0] * n + [-1] * (8 - n) and torch.equal(pages[0], want)


def test_calls_with_nothing_to_do():
    none = i32([])
    out = torch.zeros((0, 64), dtype=BF16, device=DEV)
    pages = torch.zeros((2, 1, 64, 64), dtype=BF16, device=DEV)
    masks = torch.zeros((0, 1), dtype=torch.int32, device=DEV)
    for n in (0, 2):
        ops.attention_tree(out, pages, pages, i32([[1]]), i32([0] * (n + 1)), i32([0] * n), i32([5] * n), masks, n, 1, 64, 1, 1, 64, 1.0, out)
        path, counts, nexts = ops.tree_commit(none, none, none, i32([0] * (n + 1)), i32([0] * n), i32([5] * n), n, 4, [pages[None]], i32([[1]]))
        assert path.tolist() == [[-1] * 4] * n and counts.tolist() == [0] * n and nexts.tolist() == [-1] * n
    got = ops.beam_select(torch.zeros((0, 9), device=DEV), torch.zeros((0, 3), device=DEV), 4)
    assert all(tuple(t.shape) == (0, 4) for t in got)
    ops.reorder_states([torch.zeros((3, 4), device=DEV)], i32([]).view(0, 2), i32([]).view(0, 2))
    one = torch.randn(50, device=DEV).as_strided((1, 50), (1, 1))
    check_beams(one, torch.zeros(1, 1, device=DEV), 3)


def test_beam_select_logits_of_any_size():
    """Logits too large to be scaled, rows that hold both ends, a row of one value, numbers around zero."""
    g = torch.Generator().manual_seed(0)
    big = (torch.rand(4, 9000, generator=g) * 2 - 1) * 3.3e38
    big[2] = big[2].abs()
    big[3, 1:] = -3.3e38
    check_beams(big.to(DEV), torch.zeros(2, 2, device=DEV), 8)
    tiny = (torch.rand(2, 9000, generator=g) - 0.5) * 1e-37
    check_beams(tiny.to(DEV), torch.zeros(1, 2, device=DEV), 64)


@pytest.mark.parametrize("dtype,dim", [(F32, 64), (BF16, 128)])
def test_tree_attention_one_long_context_over_all_blocks(dtype, dim):
    """One kv head and one sequence: its tiles lie on every block, and many parts are joined."""
    c = TreeCase([3], [30000], 4, 1, dim, dtype, seed=11, scale=2.0)
    c.check(c.run())
    c = TreeCase([90], [9000], 1, 1, dim, dtype, seed=12)
    c.check(c.run())


@pytest.mark.parametrize("dtype,dim", [(F32, 64), (BF16, 64), (BF16, 128), (BF16, 80)])
@pytest.mark.parametrize("scale", ["none", "tiny", "negative"])
def test_tree_attention_scales_of_any_sign(dtype, dim, scale):
    """What a node does not see stays unseen whatever scores are multiplied with."""
    rng = np.random.default_rng(3)
    sizes, pos0 = [30, 20], [100, 0]
    seen = [rng.random((n, n)) < 0.4 for n in sizes]
    seen[1][5] = False
    c = TreeCase(sizes, pos0, 4, 2, dim, dtype, seed=4, seen=seen)
    got = c.run(scale={"none": 0.0, "tiny": 1e-40, "negative": -dim ** -0.5}[scale])
    c.q = -c.q if scale == "negative" else torch.zeros_like(c.q)          # the same scores from a positive scale
    c.check(got)
    assert (got[35] == 0).all()


@pytest.mark.parametrize("nodes,dim,a_sm", [(16, 64, 2), (16, 112, 2), (16, 128, 1), (16, 256, 1), (4, 128, 2), (4, 180, 2), (4, 184, 1), (4, 256, 1)])
def test_tree_attention_has_as_many_blocks_as_the_sms_hold(nodes, dim, a_sm):
    """A job that fills the device: the scratch memory holds two partial results of 64 or 16 rows for every block that fits at a time."""
    nbytes = ops._bind().gi_attn_tree_scratch(64, nodes, 100000, 32, 8, dim, 0)
    rows = 64 if nodes == 16 else 16
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert nbytes == 4 * 68 + 2 * a_sm * sms * rows * (dim + 2) * 4


def test_tree_attention_graph_and_streams():
    """A recorded launch serves other lengths, trees and tokens; calls on two streams do not meet."""
    for dtype in (F32, BF16):
        a = TreeCase([20, 9], [300, 40], 8, 2, 128, dtype, seed=21)
        b = TreeCase([20, 9], [90, 333], 8, 2, 128, dtype, seed=22)
        pages = max(a.k.shape[0], b.k.shape[0])
        width = max(len(a.table[0]), len(b.table[0]))
        pad = lambda t: torch.cat([t, torch.zeros((pages - t.shape[0],) + tuple(t.shape[1:]), dtype=t.dtype, device=DEV)])
        rows = lambda c: i32([r + [0] * (width - len(r)) for r in c.table])
        bufs = dict(q=a.q.clone(), kcache=pad(a.k), vcache=pad(a.v), block_table=rows(a), seq_slots=i32(a.slots), seq_pos0=i32(a.pos0), masks=a.masks.clone())
        want_a, want_b = a.run(), b.run()
        out = torch.zeros_like(want_a)
        graph = torch.cuda.CUDAGraph()
        a.run(out=out, max_kv_len=400, **bufs)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            a.run(out=out, max_kv_len=400, **bufs)
        graph.replay()
        a.check(out)
        new = dict(q=b.q, kcache=pad(b.k), vcache=pad(b.v), block_table=rows(b), seq_slots=i32(b.slots), seq_pos0=i32(b.pos0), masks=b.masks)
        for name, t in new.items():
            bufs[name].copy_(t)
        graph.replay()
        b.check(out)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = [b.run() for _ in range(5)]
        here = [a.run() for _ in range(5)]
        torch.cuda.synchronize()
        assert all(torch.equal(t, want_b) for t in there) and all(torch.equal(t, want_a) for t in here)


def test_a_run_of_them_with_launches_that_begin_early():
    """Each reads what the one before it wrote; launched to begin before its predecessor has ended, eagerly and from a recording,
    the run gives what it gives with every launch on its own."""
    seqs, beams, vocab = 2, 4, 40000
    sizes, pos0 = [20, 9], [300, 40]
    case = TreeCase(sizes, pos0, 8, 2, 128, BF16, seed=31)
    logits, first_scores = randn(seqs * beams, vocab, seed=32, scale=3.0), randn(seqs, beams, seed=33)
    state0, slots = randn(seqs * beams, 4096, seed=34), i32([[3, 1, 0, 2], [6, 7, 5, 4]])
    pages0 = randn(2, 12, 2, 64, 64, dtype=BF16, seed=35)
    cu, seq_slots, at = i32([0, 20, 29]), i32([0, 1]), i32([70, 10])
    table, node_parents = i32([[1, 2, 3], [4, 5, 6]]), i32(([-1] + list(range(19))) + [-1] + list(range(8)))
    state, pages, out = state0.clone(), pages0.clone(), torch.zeros_like(case.run())

    def run():
        scores, parents, tokens = ops.beam_select(logits, first_scores, beams)
        ops.reorder_states([state], slots, parents)
        # the moved states choose which pages are copied, the beams' tokens which drafts hold
        src = (state[:2, 0] > 0).int() + 1
        ops.copy_pages([pages], src, i32_pages, i32_rows)
        case.run(out=out)
        picks = (tokens.view(-1)[0] + torch.zeros(29, dtype=torch.int32, device=DEV)).int()
        path, counts, nexts = ops.tree_commit(picks, picks.clone(), node_parents, cu, seq_slots, at, 2, 20, [pages], table)
        return [scores, parents, tokens, path, counts, nexts]

    i32_pages, i32_rows = i32([4, 5]), i32([64, 33])

    def fresh():
        state.copy_(state0)
        pages.copy_(pages0)
        out.zero_()

    was = ops.get_pdl()
    try:
        ops.set_pdl(False)
        want = [t.clone() for t in run() + [state, pages, out]]
        assert want[4].tolist() == [20, 9]                  # (every pick is every token: whole chains are accepted)
        ops.set_pdl(True)
        for _ in range(20):
            fresh()
            assert all(torch.equal(a, b) for a, b in zip(run() + [state, pages, out], want))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
        for _ in range(20):
            fresh()
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(got + [state, pages, out], want))
    finally:
        ops.set_pdl(was)


# ---- what is refused ----------------------------------------------------------------------------------------------------------
def test_refusals():
    logits, scores = randn(4, 100), torch.zeros(2, 2, device=DEV)
    for args in ((logits, scores, 0), (logits, scores, 65), (logits[:3], scores, 2), (logits.half(), scores, 2), (logits, scores.double(), 2), (logits, scores.view(-1), 2),
                 (logits.t(), torch.zeros(50, 2, device=DEV), 2), (logits[:, :2], scores, 5), (randn(65, 4), torch.zeros(1, 65, device=DEV), 2)):
        with pytest.raises(KernelError):
            ops.beam_select(*args)
    state = randn(6, 4)
    for args in (([state], i32([0, 1]), i32([0, 1])), ([state], i32([[0, 1]]), i32([[0]])), ([state.t()], i32([[0, 1]]), i32([[1, 0]])),
                 ([state, randn(5, 4)], i32([[0, 1]]), i32([[1, 0]])), ([state, state], i32([[0, 1]]), i32([[1, 0]])), ([state], i32([[0, 1]]).long(), i32([[1, 0]])),
                 ([state], i32([list(range(65))]), i32([list(range(65))])), ([state.cpu()], i32([[0, 1]]), i32([[1, 0]]))):
        with pytest.raises(KernelError):
            ops.reorder_states(*args)
    pages = randn(1, 4, 2, 64, 8)
    for args in (([pages[0]], i32([0]), i32([1])), ([pages], i32([0, 1]), i32([2])), ([pages.double()], i32([0]), i32([1])), ([pages], i32([0]), i32([1]), i32([1, 2])),
                 ([pages] * 9, i32([0]), i32([1])), ([pages.transpose(1, 2)], i32([0]), i32([1]))):
        with pytest.raises(KernelError):
            ops.copy_pages(*args)
    one = i32([0])
    for kw in (dict(max_nodes=0), dict(max_nodes=257), dict(picks=i32([0, 1])), dict(cu=i32([0])), dict(pages=[pages[0]]), dict(table=one)):
        a = dict(picks=one, tokens=one, parents=one, cu=i32([0, 1]), slots=one, pos0=one, n_seqs=1, max_nodes=1, pages=[pages], table=i32([[1]]))
        a.update(kw)
        with pytest.raises(KernelError):
            ops.tree_commit(*a.values())
    c = TreeCase([3, 4], [10, 20], 4, 2, 64, BF16)
    for kw in (dict(max_nodes=0), dict(max_nodes=257), dict(n_seqs=3), dict(masks=c.masks[:5]), dict(masks=c.masks.long()), dict(kcache=c.k.float()), dict(n_kv=3),
               dict(n_heads=8), dict(head_dim=32), dict(out=torch.zeros(7, 256, device=DEV)), dict(q=c.q[:5]), dict(max_kv_len=0), dict(max_nodes=40),
               dict(vcache=c.v[:2]), dict(cu_seqlens=c.cu.long()), dict(q=c.q.cpu())):
        with pytest.raises(KernelError):
            c.run(**kw)
