"""The operators that hold several continuations of a sequence over the paged cache, as they are measured.

A case is a dict of plain values; `op` names the operator:

* "beam": of all beams' next tokens the `width` likeliest: score + log softmax of the logits, compared in 64 bits, ties to the
  lowest beam and then the lowest token.  A logit that is no number counts as -inf.
* "states": fixed-size states of beams take their parents' place, in place, in every layer.
* "pages": the filled rows of cache pages are copied to pages of their own, keys and values of every layer.
* "tree": attention of drafted tokens, the nodes of a tree per sequence, over all cached positions and over those nodes that a
  mask of bits names.
* "commit": the walk through a tree of drafted tokens as far as the model's picks agree, and the accepted nodes' keys and values
  moved up to follow the cache directly, in every layer.

Cache sizes are those of the benchmark's Llama shapes, state sizes those of its decoders with a state.  Sequences' lengths, the
beams' parents and the trees' accepted paths belong to a case; tokens, pages, logits and numbers come from the seed.
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
PAGE = 64
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one user's beam search, one step's choice: launches and latency
        dict(name="beam_4_of_1", op="beam", seqs=1, beams=4, vocab=128256, width=8, dtype="float32"),
        # a server's beam search, 32 requests of 8 beams, twice as many candidates as beams
        dict(name="beam_8_of_32", op="beam", seqs=32, beams=8, vocab=128256, width=16, dtype="float32"),
        # 16-bit logits in rows that start on no boundary, full of equal values
        dict(name="beam_5_of_7_odd", op="beam", seqs=7, beams=5, vocab=32003, width=10, dtype="bfloat16"),
        # one user's four beams of a decoder with a matrix memory, two such layers
        dict(name="states_4", op="states", seqs=1, beams=4, layers=2, row=16 * 64 * 128),
        # eight requests of eight beams of a decoder with state-space layers
        dict(name="states_64", op="states", seqs=8, beams=8, layers=4, row=64 * 64 * 128),
        # one user's beams part: three pages, the smallest Llama shape
        dict(name="pages_3", op="pages", copies=3, layers=16, kv=8, dim=64, dtype="bfloat16"),
        # a server's beams part: 128 pages of the 3B shape
        dict(name="pages_128", op="pages", copies=128, layers=28, kv=8, dim=128, dtype="bfloat16"),
        # one user's drafted tree behind a short context
        dict(name="tree_26_ctx1500", op="tree", seqs=1, nodes_lo=26, nodes_hi=26, ctx_lo=1500, ctx_hi=1500, heads=32, kv=8, dim=128, dtype="bfloat16"),
        # a server's batch of 8 with wide trees behind long contexts
        dict(name="tree_8x64_ctx8192", op="tree", seqs=8, nodes_lo=64, nodes_hi=64, ctx_lo=8192, ctx_hi=8192, heads=32, kv=8, dim=128, dtype="bfloat16"),
        # the true 32-bit path, unequal trees and contexts
        dict(name="tree_f32_ragged", op="tree", seqs=3, nodes_lo=5, nodes_hi=17, ctx_lo=100, ctx_hi=701, heads=32, kv=8, dim=64, dtype="float32"),
        # one user's drafted tree is accepted in part
        dict(name="commit_26", op="commit", seqs=1, nodes_lo=26, nodes_hi=26, accept_lo=4, accept_hi=4, layers=16, kv=8, dim=64, dtype="bfloat16"),
        # a server's 64 trees, some of which are only the token that is fed anyway
        dict(name="commit_64x61", op="commit", seqs=64, nodes_lo=1, nodes_hi=61, accept_lo=1, accept_hi=7, layers=28, kv=8, dim=128, dtype="bfloat16"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    def spread(lo, hi):
        a, b = log_int(lo, hi), log_int(lo, hi)
        return min(a, b), max(a, b)

    op = rng.choice(["beam", "beam", "states", "pages", "tree", "tree", "tree", "commit"])
    if op == "beam":
        beams = log_int(1, 16)
        c = dict(op=op, seqs=log_int(1, 256 // max(8, beams)), beams=beams, vocab=rng.choice([128256, 32000, log_int(500, 128256)]),
                 width=rng.randint(1, 32), dtype=rng.choice(["float32", "float32", "bfloat16"]))
    elif op == "states":
        beams = log_int(1, 16)
        c = dict(op=op, seqs=log_int(1, 64 // beams), beams=beams, layers=rng.randint(1, 4), row=log_int(1000, 64 * 64 * 128))
    elif op == "pages":
        c = dict(op=op, copies=log_int(1, 128), layers=log_int(1, 28), kv=rng.choice([1, 2, 4, 8]), dim=rng.choice([40, 64, 96, 128]),
                 dtype=rng.choice(["bfloat16", "float32"]))
        if c["dtype"] == "float32":
            c["layers"] = min(c["layers"], 14)
    elif op == "tree":
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        nodes, ctx = spread(1, 100 if dtype == "bfloat16" else 24), spread(1, 12000 if dtype == "bfloat16" else 1500)
        kv, group = rng.choice([(8, 4), (8, 3), (8, 4), (4, 1), (2, 8), (5, 5)])
        most = max(1, min(32, int(8 * 64 * 8192 / max(1, nodes[1] * ctx[1]))))
        c = dict(op=op, seqs=log_int(1, most if dtype == "bfloat16" else min(8, most)), nodes_lo=nodes[0], nodes_hi=nodes[1],
                 ctx_lo=ctx[0], ctx_hi=ctx[1], heads=kv * group, kv=kv, dim=rng.choice([64, 128, 128, 80]), dtype=dtype)
    else:
        nodes, accept = spread(1, 100), spread(1, 9)
        c = dict(op=op, seqs=log_int(1, 64), nodes_lo=nodes[0], nodes_hi=nodes[1], accept_lo=accept[0], accept_hi=accept[1],
                 layers=log_int(1, 28), kv=rng.choice([2, 4, 8]), dim=rng.choice([40, 64, 128]), dtype="bfloat16")
    return c


# ---- what belongs to a case: lengths and accepted paths --------------------------------------------------------------
def _shape_rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _tree_lengths(case):
    """(nodes, cached positions) of every sequence; the ends of both ranges occur."""
    r, n = _shape_rng(case), case["seqs"]
    nodes = [r.randint(case["nodes_lo"], case["nodes_hi"]) for _ in range(n)]
    lo, hi = (case["ctx_lo"], case["ctx_hi"]) if case["op"] == "tree" else (1, 3000)
    ctx = [int(round(math.exp(r.uniform(math.log(lo), math.log(hi))))) for _ in range(n)]
    if case["op"] == "tree":
        nodes[-1], ctx[0] = case["nodes_hi"], hi
    return nodes, ctx


def _paths(case):
    """The nodes that every sequence's walk accepts: node 0 and others in ascending order."""
    r = _shape_rng(case)
    nodes, _ = _tree_lengths(case)
    out = []
    for n in nodes:
        k = min(n, r.randint(case["accept_lo"], case["accept_hi"]))
        out.append([0] + sorted(r.sample(range(1, n), k - 1)))
    return out


def _beam_parents(case):
    """Many beams go on, some are dropped in favour of a better one's second continuation."""
    r, k = _shape_rng(case), case["beams"]
    return [[j if r.random() < 0.4 else r.randrange(k) for j in range(k)] for _ in range(case["seqs"])]


def _copied_rows(case):
    r = _shape_rng(case)
    return [r.randint(1, PAGE - 1) for _ in range(case["copies"])]


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _randn(shape, dtype, g, scale=1.0):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=dtype).mul_(scale)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _trees(r, nodes, paths=None):
    """parents (-1 for a root) of every sequence's nodes, as one flat list of lists."""
    out = []
    for b, n in enumerate(nodes):
        on_path = {} if paths is None else {c: p for p, c in zip(paths[b], paths[b][1:])}
        out.append([-1 if i == 0 else on_path.get(i, r.randint(max(0, i // 2 - 3), i - 1)) for i in range(n)])
    return out


def _mask_words(parents, words):
    """Every node's ancestors and itself as bits of 32-bit words."""
    rows = []
    for tree in parents:
        seen = []
        for i, p in enumerate(tree):
            seen.append((seen[p] if p >= 0 else 0) | (1 << i))
            rows.append([(seen[i] >> (32 * w)) & 0xFFFFFFFF for w in range(words)])
    return torch.tensor([[v - (1 << 32) if v >= 1 << 31 else v for v in row] for row in rows], dtype=torch.int32).to(DEVICE)


def _offsets(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    r = random.Random(int(seed))
    op = case["op"]
    if op == "beam":
        s, k, v = case["seqs"], case["beams"], case["vocab"]
        logits = _randn((s * k, v), torch.float32, g, 3.0).to(DTYPES[case["dtype"]])
        scores = -8.0 * torch.rand((s, k), generator=g, device=DEVICE)
        return dict(op=op, logits=logits, scores=scores.sort(dim=1, descending=True).values.contiguous(), width=min(case["width"], k * v))
    if op == "states":
        s, k = case["seqs"], case["beams"]
        states = [_randn((s * k + 1, case["row"]), torch.float32, g) for _ in range(case["layers"])]
        order = list(range(s * k))
        r.shuffle(order)
        return dict(op=op, states=states, slots=_i32(order).view(s, k), parents=_i32(_beam_parents(case)))
    if op == "pages":
        n = case["copies"]
        shape = (case["layers"], 2 * n + 1, case["kv"], PAGE, case["dim"])
        pages = [_randn(shape, DTYPES[case["dtype"]], g) for _ in range(2)]
        order = list(range(1, 2 * n + 1))
        r.shuffle(order)
        return dict(op=op, pages=pages, src=_i32(order[:n]), dst=_i32(order[n:]), rows=_i32(_copied_rows(case)))
    nodes, ctx = _tree_lengths(case)
    total, dtype = sum(nodes), DTYPES[case["dtype"]]
    state = dict(op=op, cu=_i32(_offsets(nodes)), slots=_i32(list(range(case["seqs"]))), pos0=_i32(ctx), seqs=case["seqs"], max_nodes=max(nodes))
    if op == "tree":
        held = [range((c + n + PAGE - 1) // PAGE) for c, n in zip(ctx, nodes)]
    else:                                   # only the pages that hold the trees
        held = [range(c // PAGE, (c + n + PAGE - 1) // PAGE) for c, n in zip(ctx, nodes)]
    n_pages = sum(len(h) for h in held)
    order = list(range(1, n_pages + 1))
    r.shuffle(order)
    table = [[0] * (max(h.stop for h in held) + 1) for _ in held]
    for row, h in zip(table, held):
        for i in h:
            row[i] = order.pop()
    state["table"] = _i32(table)
    if op == "tree":
        h, kv, d = case["heads"], case["kv"], case["dim"]
        # the packed rows of a step (queries, then its keys and values); scores spread over a few units
        state["qkv"] = _randn((total, (h + 2 * kv) * d), torch.float32, g, 2.0).to(dtype)
        state["k"], state["v"] = (_randn((n_pages + 1, kv, PAGE, d), dtype, g) for _ in range(2))
        state["masks"] = _mask_words(_trees(r, nodes), (max(nodes) + 31) // 32)
        state |= dict(heads=h, kv=kv, dim=d, scale=d ** -0.5, max_len=max(c + n for c, n in zip(ctx, nodes)))
        return state
    paths = _paths(case)
    parents = _trees(r, nodes, paths)
    tokens, picks = [], []
    for tree, path in zip(parents, paths):
        own_tokens = [r.randrange(128256) for _ in tree]
        taken = {p: c for p, c in zip(path, path[1:])}
        for i, p in enumerate(tree):        # a sibling with an accepted node's token would be taken in its place
            while i > 0 and i != taken.get(p) and p in taken and own_tokens[i] == own_tokens[taken[p]]:
                own_tokens[i] = r.randrange(128256)
        for i in range(len(tree)):
            children = {own_tokens[c] for c, p in enumerate(tree) if p == i}
            pick = own_tokens[taken[i]] if i in taken else r.randrange(128256)
            while i not in taken and pick in children:
                pick = r.randrange(128256)
            picks.append(pick)
        tokens += own_tokens
    shape = (case["layers"], n_pages + 1, case["kv"], PAGE, case["dim"])
    state["pages"] = [_randn(shape, dtype, g) for _ in range(2)]
    state |= dict(picks=_i32(picks), tokens=_i32(tokens), parents=_i32([p for t in parents for p in t]))
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(state):
    op = state["op"]
    if own:
        from ghost_infer_b200.kernels import ops
        if op == "beam":
            return ops.beam_select(state["logits"], state["scores"], state["width"])
        if op == "states":
            ops.reorder_states(state["states"], state["slots"], state["parents"])
            return state["states"]
        if op == "pages":
            ops.copy_pages(state["pages"], state["src"], state["dst"], state["rows"])
            return state["pages"]
        if op == "tree":
            out = torch.empty((state["qkv"].shape[0], state["heads"] * state["dim"]), dtype=state["qkv"].dtype, device=state["qkv"].device)
            return ops.attention_tree(state["qkv"], state["k"], state["v"], state["table"], state["cu"], state["slots"], state["pos0"],
                                      state["masks"], state["seqs"], state["max_nodes"], state["max_len"], state["heads"], state["kv"],
                                      state["dim"], state["scale"], out)
        path, counts, nexts = ops.tree_commit(state["picks"], state["tokens"], state["parents"], state["cu"], state["slots"], state["pos0"],
                                              state["seqs"], state["max_nodes"], state["pages"], state["table"])
        return path, counts, nexts, state["pages"]
    return {"beam": _plain_beam, "states": _plain_states, "pages": _plain_pages, "tree": _plain_tree, "commit": _plain_commit}[op](state)


def _plain_beam(state):
    s, k = state["scores"].shape
    m = state["width"]
    x = state["logits"].float()
    x = torch.where(x.isnan(), float("-inf"), x)
    v = x.shape[1]
    wide = x.double()
    top = wide.amax(dim=1, keepdim=True)
    base = state["scores"].double().view(-1, 1) - (top + (wide - top).exp().sum(dim=1, keepdim=True).log())
    # a row's likeliest tokens, ties to the lowest: a whole-number key of 32 bits of value and 32 bits of distance from the end
    bits = x.view(torch.int32).long()
    bits = torch.where(bits < 0, -0x80000000 - bits, bits)
    key = bits * (1 << 32) + torch.arange(v - 1, -1, -1, device=x.device)
    best = torch.topk(key, min(m, v), dim=1, sorted=True).values
    token = v - 1 - (best & 0xFFFFFFFF)
    value = (base + wide.gather(1, token)).view(s, -1)
    value, at = torch.sort(value, dim=1, descending=True, stable=True)
    value, at = value[:, :m], at[:, :m]
    parent, token = at // min(m, v), token.view(s, -1).gather(1, at)
    none = ~torch.isfinite(value)
    return value.float(), torch.where(none, -1, parent).int(), torch.where(none, -1, token).int()


def _plain_states(state):
    slots = state["slots"].long()
    to, source = slots.view(-1), slots.gather(1, state["parents"].long()).view(-1)
    for t in state["states"]:
        t[to] = t[source]
    return state["states"]


def _plain_pages(state):
    src, dst = state["src"].long(), state["dst"].long()
    filled = torch.arange(PAGE, device=src.device)[None, :] < state["rows"][:, None]
    for t in state["pages"]:
        t[:, dst] = torch.where(filled[None, :, None, :, None], t[:, src], t[:, dst])
    return state["pages"]


def _plain_tree(state):
    h, kv, d, n = state["heads"], state["kv"], state["dim"], state["max_nodes"]
    cu, pos0, masks = state["cu"].long(), state["pos0"].long(), state["masks"]
    b, dev = state["seqs"], masks.device
    place = torch.arange(n, device=dev)
    live = place[None, :] < (cu[1:] - cu[:-1])[:, None]                       # [b, n]
    row = torch.where(live, cu[:-1, None] + place[None, :], 0)
    q = state["qkv"][:, :h * d].float()[row].view(b, n, kv, h // kv, d).permute(0, 2, 3, 1, 4)
    pages = state["table"].long()[state["slots"].long()][:, :(state["max_len"] + PAGE - 1) // PAGE]
    k, v = (state[x][pages].float().permute(0, 2, 1, 3, 4).reshape(b, kv, -1, d) for x in ("k", "v"))
    key = torch.arange(k.shape[2], device=dev)
    node = key[None, :] - pos0[:, None]                                       # [b, keys]: place in the tree, negative: cached before it
    held = node < (cu[1:] - cu[:-1])[:, None]
    word = (node.clamp(0, n - 1) // 32)[:, None, :].expand(b, n, -1)
    bit = (masks[row].gather(2, word) >> (node.clamp(0, n - 1) % 32)[:, None, :]) & 1
    seen = ((node < 0)[:, None, :] | (bit != 0)) & held[:, None, :]           # [b, n, keys]
    v = torch.where(held[:, None, :, None], v, 0.0)
    score = (q.reshape(b, kv, -1, d) @ k.transpose(2, 3)).view(b, kv, h // kv, n, -1) * state["scale"]
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    top = score.amax(dim=-1, keepdim=True)
    weight = (score - torch.where(torch.isfinite(top), top, 0.0)).exp()
    total = weight.sum(dim=-1, keepdim=True)
    out = (weight.view(b, kv, -1, weight.shape[-1]) @ v).view(b, kv, h // kv, n, d)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(b, n, h * d)
    return out[live].to(state["qkv"].dtype)


def _plain_commit(state):
    cu, pos0, n = state["cu"].long(), state["pos0"].long(), state["max_nodes"]
    dev, b = cu.device, state["seqs"]
    place = torch.arange(n, device=dev)
    size = cu[1:] - cu[:-1]
    live = place[None, :] < size[:, None]
    row = torch.where(live, cu[:-1, None] + place[None, :], 0)
    parent, token, pick = (state[x].long()[row] for x in ("parents", "tokens", "picks"))
    up = parent.clamp(min=0)
    # a node agrees if its token is its parent's pick and no sibling before it has that token
    twin = (parent[:, :, None] == parent[:, None, :]) & (token[:, :, None] == token[:, None, :]) & live[:, None, :] & (place[None, :] < place[:, None])[None]
    agrees = live & ((place == 0)[None] | ((token == pick.gather(1, up)) & ~twin.any(dim=2)))
    # who is whose ancestor, by repeated squaring of "parent or self"
    reach = torch.zeros((b, n, n), device=dev)
    reach.scatter_(2, torch.where(place[None, :] > 0, up, 0)[:, :, None], 1.0)
    reach = torch.maximum(reach, torch.eye(n, device=dev)[None])
    reach = reach @ reach
    reach = reach.clamp(max=1) @ reach.clamp(max=1)
    reach = reach.clamp(max=1) @ reach.clamp(max=1)
    reach = reach.clamp(max=1) @ reach.clamp(max=1)
    reach = reach.clamp(max=1) @ reach.clamp(max=1)
    reach = reach.clamp(max=1) @ reach.clamp(max=1)
    reach = reach.clamp(max=1) @ reach.clamp(max=1)
    reach = reach.clamp(max=1) @ reach.clamp(max=1) > 0
    taken = agrees & ~(reach & ~agrees[:, None, :]).any(dim=2)
    count = taken.sum(dim=1)
    path = torch.where(taken, place[None, :], n).sort(dim=1).values
    last = path.gather(1, (count - 1).clamp(min=0)[:, None]).clamp(max=n - 1)
    nexts = torch.where(count > 0, pick.gather(1, last)[:, 0], -1)
    on = path < n
    table = state["table"].long()[state["slots"].long()]
    fr, to = pos0[:, None] + path.clamp(max=n - 1), pos0[:, None] + place[None, :]
    fr, to = torch.where(on, fr, pos0[:, None]), torch.where(on, to, pos0[:, None])    # the rest: the root onto itself
    fr_page, to_page = table.gather(1, fr // PAGE).view(-1), table.gather(1, to // PAGE).view(-1)
    fr, to = (fr % PAGE).view(-1), (to % PAGE).view(-1)
    for t in state["pages"]:
        t[:, to_page, :, to] = t[:, fr_page, :, fr].clone()
    return torch.where(on, path, -1).int(), count.int(), nexts.int(), state["pages"]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    size = 4 if case.get("dtype", "float32") == "float32" else 2
    if op == "beam":
        rows = case["seqs"] * case["beams"]
        return {"bytes": rows * case["vocab"] * size + case["seqs"] * case["width"] * 12, "flops": 4 * rows * case["vocab"]}
    if op == "states":                      # a state that several beams take is read once; a beam that goes on needs nothing moved
        written = sum(p != j for row in _beam_parents(case) for j, p in enumerate(row))
        read = sum(len({p for j, p in enumerate(row) if p != j}) for row in _beam_parents(case))
        places = 2 * 4 * case["seqs"] * case["beams"]
        return {"bytes": places + 4 * (read + written) * case["row"] * case["layers"], "flops": 0}
    if op == "pages":
        return {"bytes": 2 * 2 * sum(_copied_rows(case)) * case["layers"] * case["kv"] * case["dim"] * size, "flops": 0}
    nodes, ctx = _tree_lengths(case)
    if op == "tree":
        read = sum(n + c for n, c in zip(nodes, ctx)) * 2 * case["kv"] * case["dim"] * size + 2 * sum(nodes) * case["heads"] * case["dim"] * size
        return {"bytes": read, "flops": 4 * case["heads"] * case["dim"] * sum(n * (c + 1) for n, c in zip(nodes, ctx))}
    moved = sum(sum(1 for i, p in enumerate(path) if i != p) for path in _paths(case))
    return {"bytes": 2 * 2 * moved * case["layers"] * case["kv"] * case["dim"] * size + sum(nodes) * 12 + case["seqs"] * (8 + 4 * max(nodes)), "flops": 0}


# ---- 64-bit values from the definitions, one sequence at a time ---------------------------------------------------------
def exact(case, seed):
    op = case["op"]
    if op == "beam":
        st = prepare(case, seed)
        s, k = st["scores"].shape
        values = []
        for i in range(s):
            log_p = torch.log_softmax(st["logits"][i * k:(i + 1) * k].double(), dim=1) + st["scores"][i].double()[:, None]
            values.append(torch.sort(log_p.reshape(-1), descending=True).values[:st["width"]])
        return torch.stack(values), None, None
    if op != "tree":
        return None                         # nothing is computed: rows are copied
    st = prepare(case, seed)
    cu, pos0, table, masks = (st[x].tolist() for x in ("cu", "pos0", "table", "masks"))
    h, kv, d = st["heads"], st["kv"], st["dim"]
    outs = []
    for i in range(st["seqs"]):
        n, c = cu[i + 1] - cu[i], pos0[i]
        at = torch.arange(c + n, device=DEVICE)
        page = torch.tensor(table[i], device=DEVICE)[at // PAGE]
        keys, values = (st[x][page, :, at % PAGE].double() for x in ("k", "v"))     # [positions, kv, d]
        seen = [[True] * c + [bool((masks[cu[i] + a][t // 32] >> (t % 32)) & 1) for t in range(n)] for a in range(n)]
        hidden = ~torch.tensor(seen, device=DEVICE)
        heads = []
        for j in range(h):
            q = st["qkv"][cu[i]:cu[i + 1], j * d:(j + 1) * d].double()
            w = (q @ keys[:, j // (h // kv)].T) * (d ** -0.5)
            w = torch.softmax(w.masked_fill(hidden, float("-inf")), dim=1)
            heads.append(w @ values[:, j // (h // kv)])
        outs.append(torch.cat(heads, dim=1))
    return torch.cat(outs)
