"""Several continuations of one sequence through the engine and the entry points, against the plain implementations: steps over trees
of drafted tokens, generation with them, beam search, on decoders with and without fixed-size states."""
import random

import numpy as np
import pytest
import torch

import ghost_infer_b200 as gi
import test_gpu_barovik as tb
import test_gpu_navalorn as tn
import test_gpu_nuzinex as tx
import test_gpu_sofopel as ts
import test_gpu_torutar as tt
import test_gpu_vavupel as tv
from branch_cases import plain_beam_select, plain_walk, random_tree
from ghost_infer_b200.engine.step import StepEntry, TreeEntry
from gpu_helpers import check_logits, make_engine, oracle, plain_logits, tokens_for

pytestmark = pytest.mark.gpu


def path_to(parents, node):
    out = []
    while node >= 0:
        out.append(node)
        node = parents[node]
    return out[::-1]


# ---- steps over trees -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_tree_steps_and_what_they_leave_behind(model_dirs, tiny_configs, name, dtype):
    """Every node's logits are those of its path; after the commit the slots go on as if only the accepted tokens had been fed."""
    d = model_dirs(name, dtype)
    eng = make_engine(d, dtype)
    assert eng.takes_trees()
    rng = random.Random(5)
    vocab = tiny_configs[name]["vocab_size"]
    prompts = [tokens_for(tiny_configs[name], n, n) for n in (61, 3, 100)]
    slots = [eng.cache.open_slot() for _ in prompts]
    eng.step([StepEntry(s, p) for s, p in zip(slots, prompts)])
    told = [list(p) for p in prompts]
    for round_, sizes in enumerate(([9, 1, 33], [1, 1, 1], [40, 5, 2])):
        entries = []
        for s, n in zip(slots, sizes):
            entries.append(TreeEntry(s, [rng.randrange(vocab) for _ in range(n)], random_tree(rng, n, 0.5)))
        step = eng.step_tree(entries)
        assert [eng.cache.length(s) for s in slots] == [len(t) for t in told]
        logits = step.logits.cpu().numpy()
        assert logits.shape == (sum(sizes), vocab)
        # picks that lead some way into each tree, whatever the model thinks
        picks, at = [], 0
        for e, so_far in zip(entries, told):
            n = len(e.tokens)
            for i in random.Random(round_).sample(range(n), min(n, 4)):
                path = path_to(e.parents, i)
                check_logits(logits[at + i:at + i + 1], plain_logits(d, so_far + [e.tokens[x] for x in path])[-1:], dtype, f"{name} node {i}")
            for i in range(n):
                children = [c for c in range(n) if e.parents[c] == i]
                picks.append(e.tokens[rng.choice(children)] if children and rng.random() < 0.8 else rng.randrange(vocab))
            at += n
        accepted = eng.commit_tree(step, torch.tensor(picks, dtype=torch.int32, device="cuda:0"))
        at = 0
        for k, (e, got) in enumerate(zip(entries, accepted)):
            n = len(e.tokens)
            path, nxt = plain_walk(picks[at:at + n], list(e.tokens), e.parents)
            assert got == [e.tokens[i] for i in path[1:]] + [nxt]
            told[k] += [e.tokens[i] for i in path]
            assert eng.cache.length(slots[k]) == len(told[k])
            at += n
        with pytest.raises(RuntimeError):
            eng.commit_tree(step, torch.tensor(picks, dtype=torch.int32, device="cuda:0"))
    # and one ordinary step more
    last = [rng.randrange(vocab) for _ in slots]
    out = eng.step([StepEntry(s, [t], [0]) for s, t in zip(slots, last)]).cpu().numpy()
    for r, (t, so_far) in enumerate(zip(last, told)):
        check_logits(out[r:r + 1], plain_logits(d, so_far + [t])[-1:], dtype, f"{name} after the trees")


def test_a_tree_step_that_is_not_committed_leaves_nothing(model_dirs, tiny_configs):
    d = model_dirs("A", "float32")
    eng = make_engine(d, "float32")
    prompt = tokens_for(tiny_configs["A"], 40, 1)
    s = eng.cache.open_slot()
    eng.step([StepEntry(s, prompt)])
    dropped = eng.step_tree([TreeEntry(s, [1, 2, 3], [-1, 0, 0])])
    out = eng.step([StepEntry(s, [9], [0])]).cpu().numpy()
    check_logits(out, plain_logits(d, prompt + [9])[-1:], "float32")
    with pytest.raises(RuntimeError):
        eng.commit_tree(dropped, torch.zeros(3, dtype=torch.int32, device="cuda:0"))


def test_only_the_latest_step_over_trees_can_be_committed(model_dirs, tiny_configs):
    """A step whose nodes' places were written again, given back or taken over by another sequence is refused, also where the slot
    is as long as it was."""
    d = model_dirs("A", "float32")
    eng = make_engine(d, "float32")
    prompt = tokens_for(tiny_configs["A"], 40, 1)
    picks = torch.full((3,), 5, dtype=torch.int32, device="cuda:0")
    s = eng.cache.open_slot()
    eng.step([StepEntry(s, prompt)])

    def drafted(tokens=(7, 5, 5)):
        return eng.step_tree([TreeEntry(s, list(tokens), [-1, 0, 1])])

    def again(step):
        with pytest.raises(RuntimeError):
            eng.commit_tree(step, picks)

    first = drafted((1, 2, 3))
    second = drafted()
    again(first)                                        # another step over trees
    eng.cache.truncate(s, 40)
    again(second)                                       # its pages went back
    third = drafted()
    other = eng.cache.fork(s)
    eng.cache.reorder([[s, other]], [[1, 0]])
    again(third)                                        # the slot holds what another one held
    fourth = drafted()
    eng.cache.close_slot(s)
    eng.cache.close_slot(other)
    again(fourth)
    s2 = eng.cache.open_slot()
    eng.step([StepEntry(s2, prompt)])
    assert s2 in (s, other)
    s = s2
    again(fourth)                                       # another sequence in the same slot
    assert eng.commit_tree(drafted(), picks) == [[5, 5, 5]] and eng.cache.length(s) == 43
    out = eng.step([StepEntry(s, [9], [0])]).cpu().numpy()
    check_logits(out, plain_logits(d, prompt + [7, 5, 5, 9])[-1:], "float32")


def test_trees_that_are_refused(model_dirs):
    eng = make_engine(model_dirs("A", "float32"), "float32")
    s = eng.cache.open_slot()
    for tokens, parents in (([1, 2], [-1, 1]), ([1, 2], [0, 0]), ([1, 2], [-1]), ([1, 2], [-1, -1]), ([], []), ([1, 999], [-1, 0]), ([1] * 257, [-1] + list(range(256)))):
        with pytest.raises(ValueError):
            eng.step_tree([TreeEntry(s, tokens, parents)])
    with pytest.raises(ValueError):
        eng.step_tree([TreeEntry(s, [1], [-1]), TreeEntry(s, [1], [-1])])
    assert eng.cache.length(s) == 0
    other = tb.engine_for(sorted(tb.CONFIGS)[0], "float32")
    assert not other.takes_trees()
    with pytest.raises(ValueError):
        other.step_tree([TreeEntry(other.cache.open_slot(), [1], [-1])])


# ---- generation with drafted tokens --------------------------------------------------------------------------------------
class Guess:
    """Drafts the true continuations (known from a plain run) with wrong tokens among them, as chains, bushes, or nothing."""

    def __init__(self, runs, vocab, seed):
        self.runs, self.vocab, self.rng = runs, vocab, random.Random(seed)

    def __call__(self, tokens, most):
        out, parents = [], []
        rest = next((r[len(tokens):] for r in self.runs if r[:len(tokens)] == list(tokens)), [])
        at = -1
        for t in rest:
            for wrong in range(self.rng.randrange(3)):
                if len(out) < most:
                    out.append(self.rng.randrange(self.vocab))
                    parents.append(at)
            if len(out) >= most or self.rng.random() < 0.15:
                break
            out.append(t)
            parents.append(at)
            at = len(out) - 1
        return out, parents


@pytest.mark.parametrize("name", ["A", "B", "D"])
def test_drafted_generation_is_greedy_generation(model_dirs, tiny_configs, name):
    d = model_dirs(name, "float32")
    llm = gi.LLM(d, dtype="float32", max_tokens=64 * 40)
    prompts = [tokens_for(tiny_configs[name], n, n) for n in (20, 3, 50, 33, 7)]
    want = llm.generate(prompts, max_new=40, temperature=0.0, batch_size=3, stop_token_ids=())
    runs = [p + r.tokens for p, r in zip(prompts, want)]
    for drafter, nodes in ((None, 32), (Guess(runs, 200, 1), 16), (Guess(runs, 200, 2), 256), (lambda t, most: ([], []), 8), (Guess(runs, 200, 3), 1)):
        got = llm.generate_drafted(prompts, max_new=40, drafter=drafter, max_nodes=nodes, batch_size=3, stop_token_ids=())
        assert [(r.tokens, r.finish_reason) for r in got] == [(r.tokens, r.finish_reason) for r in want]
        if isinstance(drafter, Guess) and nodes > 1:
            assert llm.last_stats.steps < 2 * 41
    assert llm.cache.free_pages == llm.cache.n_pages
    # stop tokens: one that the plain run comes by
    stop = [want[0].tokens[5], want[2].tokens[11]]
    want = llm.generate(prompts, max_new=40, temperature=0.0, batch_size=5, stop_token_ids=stop)
    got = llm.generate_drafted(prompts, max_new=40, drafter=Guess(runs, 200, 4), batch_size=5, stop_token_ids=stop)
    assert [(r.tokens, r.finish_reason, r.stopped_on) for r in got] == [(r.tokens, r.finish_reason, r.stopped_on) for r in want]


def test_drafted_generation_at_the_ends_of_context_and_pool(model_dirs, tiny_configs):
    d = model_dirs("A", "float32")                      # 128 positions
    prompts = [tokens_for(tiny_configs["A"], n, n) for n in (100, 20)]
    for max_tokens in (64 * 8, 64 * 3):
        llm = gi.LLM(d, dtype="float32", max_tokens=max_tokens)
        want = llm.generate(prompts, max_new=200, temperature=0.0, batch_size=2, stop_token_ids=())
        runs = [p + r.tokens for p, r in zip(prompts, want)]
        for drafter in (Guess(runs, 200, 5), None):
            got = llm.generate_drafted(prompts, max_new=200, drafter=drafter, batch_size=2, stop_token_ids=())
            if max_tokens > 64 * 3:                     # (which sequence a full pool ends first depends on the steps' sizes)
                assert [(r.tokens, r.finish_reason) for r in got] == [(r.tokens, r.finish_reason) for r in want]
            for r, run, p in zip(got, runs, prompts):
                both = min(len(r.tokens), len(run) - len(p))
                assert r.finish_reason == "capacity" and r.tokens[:both] == run[len(p):len(p) + both]
            assert llm.cache.free_pages == llm.cache.n_pages
        assert [r.finish_reason for r in llm.generate_drafted(prompts, max_new=0)] == ["length"] * 2


def test_rejected_drafts_keep_no_pages(model_dirs, tiny_configs):
    """A pool that just holds what one-token steps need is enough however many drafts are rejected."""
    d = model_dirs("D", "float32")
    llm = gi.LLM(d, dtype="float32", max_tokens=64 * 3)
    vocab = llm.engine.vocab
    prompts = [tokens_for(tiny_configs["D"], n, n) for n in (34, 60)]
    want = llm.generate(prompts, max_new=60, temperature=0.0, batch_size=2, stop_token_ids=())
    assert [r.finish_reason for r in want] == ["capacity"] * 2 and len(want[1].tokens) > 20      # (the second went on into the third page)
    run = prompts[0] + want[0].tokens

    def wrong(tokens, most):
        if tokens[:34] != prompts[0] or len(tokens) >= len(run):
            return [], []
        return [(run[len(tokens)] + 1) % vocab] * most, [-1] + list(range(most - 1))

    got = llm.generate_drafted(prompts, max_new=60, drafter=wrong, batch_size=2, stop_token_ids=())
    assert [(r.tokens, r.finish_reason) for r in got] == [(r.tokens, r.finish_reason) for r in want]
    # and step by step: a slot holds the pages of its accepted tokens, an uncommitted step's go back on demand
    eng = llm.engine
    s = eng.cache.open_slot()
    eng.step([StepEntry(s, prompts[0])])
    step = eng.step_tree([TreeEntry(s, [1] * 100, [-1] + list(range(99)))])
    assert eng.cache.free_pages == 0
    eng.commit_tree(step, torch.full((100,), 2, dtype=torch.int32, device="cuda:0"))
    assert eng.cache.length(s) == 35 and eng.cache.free_pages == 2
    eng.step_tree([TreeEntry(s, [1] * 100, [-1] + list(range(99)))])
    assert eng.cache.free_pages == 0 and eng.cache.truncate(s, 35) == 35 and eng.cache.free_pages == 2
    eng.cache.close_slot(s)


def test_drafted_generation_says_how_long_it_took(model_dirs, tiny_configs):
    llm = gi.LLM(model_dirs("A", "float32"), dtype="float32", max_tokens=64 * 40)
    prompts = [tokens_for(tiny_configs["A"], n, n) for n in (20, 3)]
    llm.generate_drafted(prompts, max_new=9, batch_size=1, stop_token_ids=())
    st = llm.last_stats
    assert st.prompt_secs > 0 and st.gen_secs > 0
    assert (st.prompt_tokens, st.gen_tokens, st.batches) == (23, 18, 2)


# ---- beam search ------------------------------------------------------------------------------------------------------------
def plain_beams(log_probs_of, prompt, beams, max_new, stop, width):
    """Beam search by the plain implementation: every beam's whole sequence is run again at every step."""
    live, done = [([], 0.0)], []
    for _ in range(max_new):
        logits = np.stack([log_probs_of(prompt + t) for t, _ in live])
        value, parent, token = (x[0] for x in plain_beam_select(logits, np.array([[s for _, s in live]]), min(width, logits.size)))
        nxt = []
        for rank, (v, p, t) in enumerate(zip(value, parent, token)):
            if len(nxt) == beams:
                break
            if t in stop:
                if rank < beams:
                    done.append((live[p][0], v, v / (len(live[p][0]) + 1)))
            else:
                nxt.append((live[p][0] + [int(t)], v))
        live = nxt
        if len(done) >= beams and max(v for _, v in live) <= min(sorted((v for _, v, _ in done), reverse=True)[:beams]):
            live = []
            break
    done += [(t, v, v / len(t)) for t, v in live]
    return sorted(done, key=lambda r: -r[2])[:beams]


@pytest.mark.parametrize("name,beams,max_new", [("A", 4, 12), ("B", 1, 6), ("C", 3, 70), ("A", 8, 5)])
def test_beam_search_against_the_plain_implementation(model_dirs, tiny_configs, name, beams, max_new):
    d = model_dirs(name, "float32")
    llm = gi.LLM(d, dtype="float32", max_tokens=64 * 60)
    cfg, w = oracle(d)
    import plain_llama as pl
    prompts = [tokens_for(tiny_configs[name], n, n + 1) for n in (30, 5, 63)][:1 if max_new > 20 else 3]
    # a stop token that comes up: the likeliest first token of one prompt, and one that does not
    stop = [int(np.argmax(plain_logits(d, prompts[-1])[-1])), 1]
    for stops in ((), stop):
        width = min(beams * (1 + max(1, len(stops))), 64)
        got = llm.beam_search(prompts, beams=beams, max_new=max_new, stop_token_ids=stops, batch_size=2)
        for p, results in zip(prompts, got):
            want = plain_beams(lambda t: pl.forward(cfg, w, t)[-1], p, beams, max_new, set(stops), width)
            assert [r.tokens for r in results] == [t for t, _, _ in want]
            for r, (_, v, score) in zip(results, want):
                # a few 1e-6 a token and 32-bit scores along the way
                assert abs(r.log_prob - v) <= 1e-4 * max(1, len(r.tokens)) and abs(r.score - score) <= 1e-4 * max(1, len(r.tokens))
        assert llm.cache.free_pages == llm.cache.n_pages and llm.cache.slots.free_slots == llm.cache.max_slots


def log_prob_by_prompt(engine, prompt, tokens):
    """Sum of the tokens' log probabilities from one prompt step over the whole sequence, and the largest |logit|."""
    s = engine.cache.open_slot()
    try:
        logits = engine.step([StepEntry(s, prompt + tokens, range(len(prompt) - 1, len(prompt) + len(tokens) - 1))]).double()
        lp = torch.log_softmax(logits, dim=1)
        return float(lp[torch.arange(len(tokens)), torch.tensor(tokens)].sum()), max(1.0, float(logits.abs().max()))
    finally:
        engine.cache.close_slot(s)


def recurrent_engines():
    for name in sorted(tb.CONFIGS):
        yield "barovik " + name, lambda name=name: tb.engine_for(name, "float32", max_tokens=64 * 60)
    for what, module in (("navalorn", tn), ("nuzinex", tx), ("sofopel", ts), ("torutar", tt), ("vavupel", tv)):
        for name in sorted(module.CONFIGS):
            yield f"{what} {name}", lambda module=module, name=name: module.engine_for(name, "float32", max_tokens=64 * 60)


@pytest.mark.parametrize("which,make", list(recurrent_engines()), ids=lambda x: x if isinstance(x, str) else "")
def test_beams_of_decoders_with_states(which, make):
    """States, windows and chunks follow their beams: every result's probability is that of its tokens read as a prompt."""
    from ghost_infer_b200.engine.beams import BeamSearch
    eng = make()
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, eng.vocab, size=n).tolist() for n in (37, 6)]
    got = BeamSearch(eng, 5, batch_size=2).run(prompts, 30)
    for p, results in zip(prompts, got):
        assert len(results) == 5 and len({tuple(r.tokens) for r in results}) == 5
        assert all(a.score >= b.score for a, b in zip(results, results[1:]))
        for r in results:
            assert len(r.tokens) == 30
            want, scale = log_prob_by_prompt(eng, p, r.tokens)
            # a 32-bit logit is off by up to 3e-5 of the largest one, on both sides, and so is the log of its row's sum
            assert abs(want - r.log_prob) <= 30 * 4 * 3e-5 * scale
    assert eng.cache.free_pages == eng.cache.n_pages


def test_beams_in_16_bits_share_pages(model_dirs, tiny_configs):
    """A pool that holds the prompt once and a page or two for each beam is enough."""
    d = model_dirs("D", "bfloat16")
    llm = gi.LLM(d, dtype="bfloat16", max_tokens=64 * (8 + 2 * 6 + 2), max_seq_len=1024)
    prompt = tokens_for(tiny_configs["D"], 64 * 8 - 10, 4)
    results = llm.beam_search([prompt], beams=6, max_new=40, stop_token_ids=())[0]
    assert len(results) == 6 and all(len(r.tokens) == 40 for r in results)
    for r in results:
        want, scale = log_prob_by_prompt(llm.engine, prompt, r.tokens)
        # a 16-bit logit is off by up to 2.5% of the largest one
        assert abs(want - r.log_prob) <= 40 * 4 * 0.025 * scale
    assert llm.cache.free_pages == llm.cache.n_pages


def test_command_line(model_dirs, tiny_configs, capsys):
    from ghost_infer_b200 import cli
    d = model_dirs("A", "float32")
    prompts = [tokens_for(tiny_configs["A"], n, n) for n in (9, 4)]
    text = ";".join(",".join(map(str, p)) for p in prompts)
    cli.cmd_run(cli.parse_opts([d, "-p", text, "-n", "7", "-t", "0", "--dtype", "float32"]))
    greedy = capsys.readouterr().out
    cli.cmd_run(cli.parse_opts([d, "-p", text, "-n", "7", "--draft", "8", "--dtype", "float32"]))
    assert capsys.readouterr().out == greedy
    cli.cmd_run(cli.parse_opts([d, "-p", text, "-n", "7", "--beams", "3", "--dtype", "float32"]))
    lines = capsys.readouterr().out.splitlines()
    llm = gi.LLM(d, dtype="float32", max_tokens=64 * 20)
    assert [[int(t) for t in line.split()] for line in lines] == [r[0].tokens for r in llm.beam_search(prompts, beams=3, max_new=7)]
