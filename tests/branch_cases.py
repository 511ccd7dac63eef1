"""Plain statements of the operators that hold several continuations of a sequence, in 64 bits and without the library: beam
search's choice, the walk through a tree of drafted tokens, attention over a tree.  Shared by the host and the GPU tests."""
import math
import random

import numpy as np
import torch


def plain_beam_select(logits, scores, width):
    """(scores float64, parents, tokens) as lists of rows; logits [seqs * beams, vocab] and scores [seqs, beams] are numpy float64."""
    seqs, beams = scores.shape
    vocab = logits.shape[1]
    out = []
    for s in range(seqs):
        value = np.full((beams, vocab), -np.inf)
        for j in range(beams):
            x = logits[s * beams + j].copy()
            x[np.isnan(x)] = -np.inf
            top = x.max()
            if not np.isfinite(top) or not np.isfinite(scores[s, j]):
                continue
            value[j] = (scores[s, j] - (top + math.log(np.exp(x - top).sum()))) + x
        flat = value.reshape(-1)
        # descending; of equal ones the lowest beam's first, then the larger logit (whose sum 64 bits may not tell apart), then the
        # lowest token; -0 and 0 are equal
        x = np.nan_to_num(logits[s * beams:(s + 1) * beams], nan=-np.inf, posinf=np.inf, neginf=-np.inf).reshape(-1) + 0.0
        place = np.arange(flat.size)
        order = np.lexsort((place % vocab, -x, place // vocab, -flat))[:width]
        none = ~np.isfinite(flat[order])
        out.append((flat[order], np.where(none, -1, order // vocab), np.where(none, -1, order % vocab)))
    return tuple(np.stack([row[i] for row in out]) for i in range(3))


def plain_walk(picks, tokens, parents):
    """(path, next token) of one tree."""
    if not tokens:
        return [], -1
    path = [0]
    while True:
        at = path[-1]
        child = next((i for i in range(at + 1, len(tokens)) if parents[i] == at and tokens[i] == picks[at]), None)
        if child is None:
            return path, picks[at]
        path.append(child)


def random_tree(rng, n, depth_bias=0.5):
    """Parents of n nodes, -1 for the first."""
    return [-1 if i == 0 else (i - 1 if rng.random() < depth_bias else rng.randrange(i)) for i in range(n)]


def ancestors(parents):
    """bool [n, n]: which nodes a node sees (its ancestors and itself)."""
    n = len(parents)
    seen = np.zeros((n, n), dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


def mask_words(seen_of_trees, words):
    """int32 [tokens, words] from a list of bool [n, n]."""
    rows = []
    for seen in seen_of_trees:
        for row in seen:
            bits = sum(1 << i for i, on in enumerate(row) if on)
            rows.append([(bits >> (32 * w)) & 0xFFFFFFFF for w in range(words)])
    return torch.from_numpy(np.array(rows, dtype=np.uint32).reshape(-1, words).view(np.int32).copy())


def plain_tree_attention(q, k, v, seen, scale):
    """One sequence in float64: q [n, H, d], k and v [positions, KV, d], seen bool [n, positions].  Returns (out [n, H, d],
    mean |v| under the weights [n, H, d], largest sum |q_i k_i| of a score)."""
    n, h, d = q.shape
    kv = k.shape[1]
    out, spread, most = np.zeros((n, h, d)), np.zeros((n, h, d)), 0.0
    for j in range(h):
        kj, vj = k[:, j // (h // kv)], v[:, j // (h // kv)]
        for i in range(n):
            on = np.flatnonzero(seen[i])
            if on.size == 0:
                continue
            s = kj[on] @ q[i, j] * scale
            most = max(most, float((np.abs(kj[on]) @ np.abs(q[i, j])).max()) * scale)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, j], spread[i, j] = w @ vj[on], w @ np.abs(vj[on])
    return out, spread, most
