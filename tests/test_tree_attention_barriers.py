"""The tcgen05 tree attention's barriers, every order of events tried on the CPU.

The kernel's parts (two threads that load, two that issue products, warps of both halves of the keys) are restated as lists of waits and
actions; loads and products complete at any time after they are issued, those of one issuing thread in their order.  Every wait's
barrier and parity are read from the kernel's source.  An mbarrier knows only its phase's parity: a wait passes where the number of
completed phases has the other parity."""
import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ghost_infer_b200", "csrc", "attention_tree_t5.cu")
ROLES = ("load", "score", "output", "rows")
STARTS = ("if (warp == 8 || warp == 11) {", "} else if (warp == 9) {", "} else if (warp == 10) {", "// ---- one query row and one half")


def waits_of_source():
    """{role: [(barrier, index expression, parity expression)] in the source's order}."""
    text = open(SOURCE).read()
    text = text[text.index("attn_tree_t5_kernel(const __grid_constant__"):]
    at = [text.index(s) for s in STARTS] + [text.index("tcgen05.dealloc")]
    out = {}
    for role, a, b in zip(ROLES, at, at[1:]):
        found = []
        for bar, parity in re.findall(r"mbar_wait\((.+?), \(uint32_t\)\((.+?)\), \d, &g_tree_status\)", text[a:b]):
            name, _, offset = bar.partition(" + ")
            found.append((name, offset.replace("8 * ", "1 * ").replace("16 * ", "2 * ").replace("+ 8", "+ 1"), parity))
        assert len(found) == text[a:b].count("mbar_wait(") > 0
        out[role] = found
    return out


def test_the_source_has_the_waits_that_the_search_walks_through():
    names = {role: [name for name, _, _ in found] for role, found in waits_of_source().items()}
    assert names == {"load": ["q_empty", "empty", "q_full", "full"], "score": ["q_full", "k_full", "sp_empty"],
                     "output": ["v_full", "p_full", "p_full"], "rows": ["s_full", "sp_empty", "v_full", "scanned", "zeroed", "met", "sp_empty"]}


def wait_at(source, role, n, prefix="", **env):
    name, index, parity = source[role][n]
    value = lambda text: eval(text.replace("&&", " and ").replace("/", "//"), env)
    return ("wait", (prefix + name, value(index) if index else 0), value(parity))


def programs(source, units, in_tree, stages, rescales):
    """`units`: tiles of each unit; `in_tree`: numbers of the tiles that need care."""
    def load(kind):
        prog, j = [], 0
        for f, tiles in enumerate(units):
            if kind == "K":
                if f > 0:
                    prog.append(wait_at(source, "load", 0, f=f))
                prog.append(("issue", ("Q", f)))
            for _ in range(tiles):
                if j >= stages:
                    prog.append(wait_at(source, "load", 1, kind.lower() + "_", j=j, s=j % stages, STAGES=stages))
                prog.append(("issue", (kind, j)))
                j += 1
        return prog

    scores, outputs, rows, j = [], [], ([], []), 0
    for f, tiles in enumerate(units):
        scores.append(wait_at(source, "score", 0, f=f))
        for t in range(tiles):
            env = dict(j=j, f=f, s=j % stages, buf=j & 1, STAGES=stages)
            scores.append(wait_at(source, "score", 1, **env))
            if j >= 2:
                scores.append(wait_at(source, "score", 2, **env))
            scores.append(("issue", ("S", j)))
            outputs.append(wait_at(source, "output", 0, **env))
            for half in (0, 1):
                if t == 0 and half == 0:
                    outputs.append(wait_at(source, "output", 1, **env))
                outputs += [wait_at(source, "output", 2, half=half, **env), ("issue", ("O", 2 * j + half))]
            for half in (0, 1):
                prog = rows[half]
                prog += [wait_at(source, "rows", 0, **env), ("read scores", j)]
                if t > 0 and rescales:
                    prog += [wait_at(source, "rows", 1, **env), ("rescale", j)]
                prog.append(("write weights", j))
                if j in in_tree:
                    env["in_tree_tiles"] = sorted(in_tree).index(j)
                    prog += [wait_at(source, "rows", 2, **env), ("scan", j), ("arrive", ("scanned", 0)), wait_at(source, "rows", 3, **env),
                             ("zero", j), ("arrive", ("zeroed", 0)), wait_at(source, "rows", 4, **env)]
                prog.append(("arrive", ("p_full", 2 * (j & 1) + half)))
            j += 1
        for half in (0, 1):
            rows[half].extend([("write stats", f), ("arrive", ("met", 0)), wait_at(source, "rows", 5, f=f), wait_at(source, "rows", 6, j=j),
                               ("read output", f)])
    return [load("K"), load("V"), scores, outputs, *rows]


def first_fault(units, in_tree, stages, source, rescales=True):
    """What goes wrong in some order of events, or None.  One warp for each half of the keys."""
    progs = programs(source, units, in_tree, stages, rescales)
    unit_of = [f for f, tiles in enumerate(units) for _ in range(tiles)]
    starts = [sum(units[:f]) for f in range(len(units))]
    last = {s + n - 1: f for f, (s, n) in enumerate(zip(starts, units))}
    care = sorted(in_tree)
    # memory: tiles of keys and values by stage, queries, scores' buffers by half, outputs by half (unit, tiles), flags, statistics
    memory = tuple(sorted({**{("K", s): None for s in range(stages)}, **{("V", s): None for s in range(stages)}}.items()))
    start = (tuple(0 for _ in progs), frozenset(), (), memory)
    seen, todo = {start}, [start]
    while todo:
        at, flying, arrivals, memory = todo.pop()
        count, mem = dict(arrivals), dict(memory)
        need = {"scanned": 2, "zeroed": 2, "met": 2}
        after = []

        def push(at, flying, count, mem):
            after.append((at, flying, tuple(sorted(count.items())), tuple(sorted(mem.items()))))

        for i, prog in enumerate(progs):
            if at[i] == len(prog):
                continue
            op, half = prog[at[i]], i - 4
            moved = at[:i] + (at[i] + 1,) + at[i + 1:]
            what, j = op[0], op[1]
            if what == "wait":
                if count.get(j, 0) // need.get(j[0], 1) & 1 != op[2]:
                    push(moved, flying, count, mem)
                continue
            new = dict(mem)
            if what == "issue":
                if j[0] in "KV":
                    new[(j[0], j[1] % stages)] = None          # from now on anything
                elif j[0] == "Q":
                    new[("Q", 0)] = None
                push(moved, flying | {j}, count, new)
                continue
            if what == "arrive":
                push(moved, flying, {**count, j: count.get(j, 0) + 1}, mem)
                continue
            if what == "read scores":
                if mem.get(("S", 2 * (j & 1) + half)) != ("scores", j):
                    return f"scores of tile {j} read from {mem.get(('S', 2 * (j & 1) + half))}"
            elif what == "rescale":
                if mem.get(("O", half)) != (unit_of[j], j - starts[unit_of[j]]):
                    return f"outputs rescaled at tile {j} with {mem.get(('O', half))} added"
            elif what == "write weights":
                new[("S", 2 * (j & 1) + half)] = ("weights", j)
            elif what == "scan":
                if mem[("V", j % stages)] != (j, 0):
                    return f"values of tile {j} scanned in {mem[('V', j % stages)]}"
                kept = ("flags", care.index(j) & 1)
                new[kept] = tuple(sorted({*mem.get(kept, ()), j}))
            elif what == "zero":
                kept = ("flags", care.index(j) & 1)
                if mem.get(kept) != (j,):
                    return f"flags of tile {j} are those of {mem.get(kept)}"
                tile, zeroed = mem[("V", j % stages)] or (None, 0)
                if tile != j:
                    return f"values of tile {j} zeroed in {tile}"
                new[("V", j % stages)] = (j, zeroed + 1)
                if half == 0:
                    new[("flags", care.index(j) + 1 & 1)] = ()
            elif what == "write stats":
                new[("stats", 2 * (j & 1) + half)] = j
            elif what == "read output":
                if mem.get(("stats", 2 * (j & 1) + (half ^ 1))) != j:
                    return "statistics of another unit"
                if any(mem.get(("O", h)) != (j, units[j]) for h in (0, 1)):
                    return f"outputs of unit {j} read as {mem.get(('O', 0))}, {mem.get(('O', 1))}"
            push(moved, flying, count, new)
        for event in flying:                                   # something completes
            kind, j = event
            new, bars = dict(mem), []
            if kind in "SO" and (kind, j - 1) in flying:
                continue                                       # one issuing thread's products run in their order
            if kind == "Q":
                new[("Q", 0)], bars = j, [("q_full", 0)]
            elif kind in "KV":
                new[(kind, j % stages)], bars = (j if kind == "K" else (j, 0)), [(kind.lower() + "_full", j % stages)]
            elif kind == "S":
                if mem[("K", j % stages)] != j or mem.get(("Q", 0)) != unit_of[j]:
                    return f"scores of tile {j} from keys {mem[('K', j % stages)]} and queries {mem.get(('Q', 0))}"
                for h in (0, 1):
                    new[("S", 2 * (j & 1) + h)] = ("scores", j)
                bars = [("s_full", j & 1), ("k_empty", j % stages)] + ([("q_empty", 0)] if j in last else [])
            else:
                h, j = j & 1, j >> 1
                f = unit_of[j]
                if mem.get(("S", 2 * (j & 1) + h)) != ("weights", j):
                    return f"outputs of tile {j} from {mem.get(('S', 2 * (j & 1) + h))}"
                if mem[("V", j % stages)] != (j, 2 if j in in_tree else 0):
                    return f"outputs of tile {j} from values {mem[('V', j % stages)]}"
                new[("O", h)] = (f, 1) if j == starts[f] else (f, mem[("O", h)][1] + 1)
                bars = [("sp_empty", j & 1), ("v_empty", j % stages)] if h else []
            more = dict(count)
            for b in bars:
                more[b] = more.get(b, 0) + 1
            push(at, flying - {event}, more, new)
        if not after and any(p < len(prog) for p, prog in zip(at, progs)):
            return "all wait for one another"
        for state in after:
            if state not in seen:
                seen.add(state)
                todo.append(state)
    return None


CASES = [((1,), {0}), ((2,), {1}), ((3,), {2}), ((1, 1), {0, 1}), ((1, 1), set()), ((2, 1), {2}), ((1, 2), {0}), ((1, 1, 1), {0, 1, 2}), ((3,), {1, 2})]


@pytest.mark.parametrize("rescales", [True, False])
@pytest.mark.parametrize("stages", [2, 4])
@pytest.mark.parametrize("units, in_tree", CASES, ids=str)
def test_no_order_of_events_reads_or_overwrites_the_wrong_numbers(units, in_tree, stages, rescales):
    assert first_fault(units, in_tree, stages, waits_of_source(), rescales) is None


@pytest.mark.parametrize("role, n, units, in_tree, rescales", [
    ("load", 0, (1, 1), {0}, False), ("load", 1, (3,), {2}, False), ("score", 2, (3,), {2}, False), ("output", 1, (1, 1), set(), False),
    ("rows", 1, (2,), {1}, True), ("rows", 3, (1,), {0}, False), ("rows", 5, (1,), set(), False), ("rows", 6, (1,), set(), False)])
def test_the_search_finds_out_where_a_wait_is_gone(role, n, units, in_tree, rescales):
    without = waits_of_source()
    without[role][n] = ("nobody", "", "1")                 # the phase before the first: passes at once
    assert first_fault(units, in_tree, 2, without, rescales) is not None
