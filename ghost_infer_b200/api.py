"""The Python entry point: load a model folder, generate from token-id prompts.

    from ghost_infer_b200 import LLM
    llm = LLM("model_dir", dtype="bfloat16", max_tokens=8 * 4096)
    results = llm.generate([[1, 5, 9], [4, 4]], max_new=16, temperature=0.0)

Option names and defaults are the reference's command line's (src/main.rs:55-65): max_new 256,
temperature 0.7 (0 = greedy), top_k 40 (0 = all), top_p 0.9, seed from the clock.  Prompts are token
ids: the tokenizer is not part of this library.
"""
from __future__ import annotations

from typing import List, Mapping, Optional, Sequence

from .engine.beams import BeamResult, BeamSearch
from .engine.drafted import DraftedLoop, PromptLookup
from .engine.generate import GenerationLoop, GenerationResult, GenerationStats
from .engine.model import Model
from .engine.step import Engine
from .sampling import DeviceSampler, SamplingParams


class LLM:
    def __init__(self, model, dtype: str = "bfloat16", device: str = "cuda:0", max_tokens: int = 8 * 2048,
                 max_slots: Optional[int] = None, max_seq_len: Optional[int] = None, seed: int = 0,
                 beyond_trained_positions: bool = False):
        """`model`: a model folder (config.json, model.safetensors), or a config mapping, for which random
        weights are made on the device from `seed`.  `max_seq_len` above the model's own
        `max_position_embeddings` is lowered to it unless `beyond_trained_positions` is set."""
        if isinstance(model, Model):
            self.model = model
        elif isinstance(model, Mapping):
            self.model = Model.random(model, seed=seed, dtype=dtype, device=device)
        else:
            self.model = Model.from_pretrained(str(model), dtype=dtype, device=device)
        self.cache = self.model.new_cache(max_tokens=max_tokens, max_slots=max_slots, max_seq_len=max_seq_len,
                                          beyond_trained_positions=beyond_trained_positions)
        self.engine = Engine(self.model, self.cache)
        self.last_stats: Optional[GenerationStats] = None

    @property
    def stop_token_ids(self) -> Sequence[int]:
        return tuple(self.model.spec.stop_token_ids)

    def generate(self, prompts: Sequence[Sequence[int]], max_new: int = 256, temperature: float = 0.7,
                 top_k: int = 40, top_p: float = 0.9, seed: Optional[int] = None,
                 stop_token_ids: Optional[Sequence[int]] = None, batch_size: int = 8,
                 on_token=None, max_step_tokens: Optional[int] = None,
                 time_steps_every: Optional[int] = None) -> List[GenerationResult]:
        """Generates for every prompt, `batch_size` at a time, one batch after another.  `max_step_tokens`
        bounds the prompt tokens a single step carries (long prompts are then read in several steps).
        `time_steps_every` = n records the device time of every stretch of n decode steps in `last_stats.step_ms`."""
        params = SamplingParams(temperature=temperature, top_k=top_k, top_p=top_p, seed=seed)
        sampler = DeviceSampler(params, self.model.rt.device)
        stop = self.stop_token_ids if stop_token_ids is None else stop_token_ids
        loop = GenerationLoop(self.engine, sampler, stop_token_ids=stop, batch_size=batch_size, on_token=on_token,
                              max_step_tokens=max_step_tokens, time_steps_every=time_steps_every)
        results = loop.run(prompts, max_new)
        self.last_stats = loop.stats
        self._check_kernels()
        return results

    def _check_kernels(self) -> None:
        if self.model.rt.device.type == "cuda":
            from .kernels import ops
            ops.check_status()          # a kernel whose bounded wait ran out has said so: never hand out its tokens silently

    def beam_search(self, prompts: Sequence[Sequence[int]], beams: int = 4, max_new: int = 256, length_penalty: float = 1.0,
                    stop_token_ids: Optional[Sequence[int]] = None, batch_size: int = 1) -> List[List[BeamResult]]:
        """The `beams` (1 to 32) best continuations of every prompt that beam search finds, best first, `batch_size` prompts at a
        time.  Results are ordered by log probability / tokens ** length_penalty; a search ends when as many results have
        ended as there are beams and nothing still going is more probable than the `beams`-th most probable of them, or at `max_new`
        tokens.  That end goes by log probability alone: with a penalty above zero a longer result may have had a better
        score than those found, and is not looked for."""
        stop = self.stop_token_ids if stop_token_ids is None else stop_token_ids
        out = BeamSearch(self.engine, beams, stop, length_penalty, batch_size).run(prompts, max_new)
        self._check_kernels()
        return out

    def generate_drafted(self, prompts: Sequence[Sequence[int]], max_new: int = 256, drafter=None, max_nodes: int = 32,
                         stop_token_ids: Optional[Sequence[int]] = None, batch_size: int = 8) -> List[GenerationResult]:
        """`generate` at temperature 0, several tokens a step where a draft is right.  `drafter(tokens, most)` gives at most `most`
        tokens that may follow and, for each, which of them it continues (-1: the last of `tokens`); None: `PromptLookup`, what
        followed the same words earlier in the sequence.  `max_nodes` (1 to 256): tokens a sequence runs in one step.  For models
        that attend to all cached positions in every layer.  A step over trees is launched kernel by kernel where `generate` replays a
        recording, so it takes several times as long: it pays where enough drafted tokens are right."""
        stop = self.stop_token_ids if stop_token_ids is None else stop_token_ids
        loop = DraftedLoop(self.engine, drafter if drafter is not None else PromptLookup(), stop, batch_size, max_nodes)
        results = loop.run(prompts, max_new)
        self.last_stats = loop.stats
        self._check_kernels()
        return results
