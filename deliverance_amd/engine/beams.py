"""Beam search: the most likely continuations of a prompt, by summed log-probability.

Every prompt has ``num_beams`` beams, each a request of the cache manager.  A step runs one token of every beam of every prompt;
``ops.beam_select`` chooses among all beams and the vocabulary; a beam that is continued keeps its place, the places of the others
go to what continues it: the cache manager shares the full pages (``CacheManager.reorder``) and ``ops.state_reorder`` copies
what a beam holds for itself, the page that is being written and its recurrent states.  Layers of softmax attention without extras (those that go
through ``ops.paged_attention``) read the pages that a prompt's beams have in common once for all of them where that is ahead (``ops.attention_beams``);
the other designs' attention and latent rows are read beam by beam.

``BeamGroup`` is the host's part of the search for one prompt and sees candidates only; ``BeamSearch`` drives the engine.
"""
from __future__ import annotations

import math
import time
from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..kernels import ops
from ..profiler import InferenceProfiler
from .step import BeamStep, StepEntry


@dataclass
class BeamParameters:
    """``num_beams`` continuations of up to ``max_tokens`` tokens (``ntokens`` bounds prompt + generated positions, as in
    ``GeneratorParameters``); hypotheses are ranked by score / length ** ``length_penalty`` (-32 to 32; length: generated tokens).  The search of a
    prompt ends when it has ``num_beams`` finished hypotheses and no live beam's score / length ** ``length_penalty`` is better than
    the worst of them, or, with ``early_stopping``, as soon as it has them."""
    num_beams: int = 4
    max_tokens: Optional[int] = None
    ntokens: Optional[int] = None
    length_penalty: float = 1.0
    early_stopping: bool = False
    ignore_eos: bool = False

    def validate(self, n_ends: int) -> None:
        if not 1 <= self.num_beams <= ops.MAX_BEAMS:
            raise ValueError(f"num_beams must be in 1..{ops.MAX_BEAMS}")
        if self.candidates(n_ends) > ops.MAX_CANDIDATES:
            raise ValueError(f"{self.num_beams} beams with {n_ends} end tokens: at most {ops.MAX_CANDIDATES} candidates a step")
        if self.max_tokens is not None and self.max_tokens <= 0:
            raise ValueError("max_tokens must be positive")
        if self.ntokens is not None and self.ntokens <= 0:
            raise ValueError("ntokens must be positive")
        if not abs(self.length_penalty) <= 32:             # (the power of a length must be a number, and not 0)
            raise ValueError("length_penalty must be in -32..32")

    def candidates(self, n_ends: int) -> int:
        """So many that ``num_beams`` of them go on, whichever end."""
        return self.num_beams * (1 if self.ignore_eos else 1 + n_ends)


@dataclass
class BeamHypothesis:
    tokens: List[int]
    score: float                        # the tokens' summed log-probability
    rank: float                         # score / len(tokens) ** length_penalty
    finish_reason: str                  # "stop" | "length"


@dataclass
class BeamResponse:
    hypotheses: List[BeamHypothesis] = field(default_factory=list)      # best first
    prompt_tokens: int = 0
    total_time_ms: float = 0.0

    @property
    def generated_tokens(self) -> List[int]:
        return self.hypotheses[0].tokens if self.hypotheses else []


class BeamGroup:
    """The beams of one prompt: what they have generated, their scores, and the hypotheses that are finished."""

    def __init__(self, params: BeamParameters, ends, max_new: int):
        self.params, self.max_new = params, max_new
        self.ends = frozenset() if params.ignore_eos else frozenset(ends)
        B = params.num_beams
        self.tokens: List[List[int]] = [[] for _ in range(B)]
        self.scores: List[float] = [0.0] + [-math.inf] * (B - 1)          # one beam, the prompt's, until the first choice
        self.finished: List[BeamHypothesis] = []
        self.done = False

    def _finish(self, tokens: List[int], score: float, reason: str) -> None:
        self.finished.append(BeamHypothesis(tokens, score, score / len(tokens) ** self.params.length_penalty, reason))
        self.finished.sort(key=lambda h: -h.rank)                         # (stable: the earlier of equal ones stays in front)
        del self.finished[self.params.num_beams:]

    def take(self, candidates: Sequence[Tuple[float, int, int]]) -> List[int]:
        """One choice's candidates (score, parent, token), best first; returns the parent of every place."""
        B = self.params.num_beams
        goes_on: List[Tuple[float, int, int]] = []
        for rank, (score, parent, token) in enumerate(candidates):
            if token < 0 or len(goes_on) == B:
                break
            if token in self.ends:
                if rank < B:                                              # (an end that num_beams others beat is not one of the best)
                    self._finish(self.tokens[parent] + [token], score, "stop")
            else:
                goes_on.append((score, parent, token))
        # who is continued keeps its place for the first that continues it; the others get the places that are free
        place_of, rest = {}, []
        for c in goes_on:
            if c[1] in place_of:
                rest.append(c)
            else:
                place_of[c[1]] = c
        free = [b for b in range(B) if b not in place_of]
        place_of.update(zip(free, rest))
        parents = [place_of[b][1] if b in place_of else b for b in range(B)]
        self.tokens = [self.tokens[place_of[b][1]] + [place_of[b][2]] if b in place_of else self.tokens[b] + [0] for b in range(B)]
        self.scores = [place_of[b][0] if b in place_of else -math.inf for b in range(B)]
        n = len(self.tokens[0])
        if not goes_on:
            self.done = True
        elif n >= self.max_new:
            for score, tokens in zip(self.scores, self.tokens):
                if score > -math.inf:
                    self._finish(tokens, score, "length")
            self.done = True
        elif len(self.finished) == B:
            self.done = self.params.early_stopping or self.finished[-1].rank >= max(self.scores) / n ** self.params.length_penalty
        return parents


class _Live:
    """A prompt that is being searched: its requests in the cache, and the positions that its beams' tables share, per group."""

    def __init__(self, index: int, group: BeamGroup, n_beams: int, n_groups: int, prompt: List[int]):
        self.index, self.group, self.prompt = index, group, prompt
        self.rids = [("beam", index, b) for b in range(n_beams)]
        self.shared_pages = [0] * n_groups
        self.t_start = time.perf_counter()


class BeamSearch:
    def __init__(self, cache, runner, config, engine_config, params: BeamParameters):
        self.cache, self.mgr, self.runner, self.config = cache, cache.manager, runner, config
        self.engine_config, self.params = engine_config, params
        self.ends = set(config.eos_token_ids)
        params.validate(len(self.ends))
        self.n_keep = params.candidates(len(self.ends))
        if params.num_beams > engine_config.max_num_seqs:
            raise ValueError(f"{params.num_beams} beams, the engine takes {engine_config.max_num_seqs} sequences")
        if self.mgr.n_state_slots and params.num_beams > self.mgr.n_state_slots:
            raise ValueError(f"{params.num_beams} beams, the engine has {self.mgr.n_state_slots} state slots")

    # ---- what a prompt needs ------------------------------------------------------------------
    def _max_new(self, prompt: Sequence[int]) -> int:
        """As for a sampled request: the last generated token may stand at position ``ntokens``, which is never computed."""
        limit = self.config.max_positions if self.params.ntokens is None else self.params.ntokens
        if limit > self.config.max_positions:
            raise ValueError(f"ntokens {limit} exceed config length {self.config.max_positions}")
        if not prompt or len(prompt) >= limit:
            raise ValueError(f"a prompt of {len(prompt)} tokens, ntokens {limit}")
        for t in prompt:
            if not (0 <= int(t) < self.config.vocab_size):
                raise ValueError(f"token id {t} is outside the vocabulary of {self.config.vocab_size}")
        n = limit - len(prompt) + 1
        return n if self.params.max_tokens is None else min(n, self.params.max_tokens)

    def _pages(self, n_prompt: int, max_new: int) -> int:
        """Pages per cache group that a prompt's beams never exceed: the prompt's full ones once, all others a beam each (the
        last token that is computed is the one before the last generated)."""
        ps = self.mgr.page_size
        shared = n_prompt // ps
        return shared + self.params.num_beams * (-(-(n_prompt + max_new - 1) // ps) - shared)

    # ---- the search -----------------------------------------------------------------------------
    def run(self, prompts: Sequence[Sequence[int]]) -> List[BeamResponse]:
        B = self.params.num_beams
        waiting = []
        for i, p in enumerate(prompts):
            p = [int(t) for t in p]
            n = self._max_new(p)
            need = self._pages(len(p), n)
            if any(need > pool.n_pages for pool in self.mgr.pools):
                raise ValueError(f"{B} beams of {len(p)} + {n} tokens need {need} pages of {self.mgr.page_size} tokens, "
                                 f"the pool has {min(pool.n_pages for pool in self.mgr.pools)}")
            waiting.append((i, p, n, need))
        out: List[Optional[BeamResponse]] = [None] * len(prompts)
        live: List[_Live] = []
        held: Dict[int, int] = {}                          # prompt -> pages that are kept free for it
        try:
            while waiting or live:
                new = []
                while waiting and self._room(waiting[0][3], held, len(live) + len(new)):
                    i, p, n, need = waiting.pop(0)
                    held[i] = need
                    new.append(_Live(i, BeamGroup(self.params, self.ends, n), B, len(self.cache.groups), p))
                if new:
                    live += new
                    with InferenceProfiler.timer("beam_search.prompts"):
                        self._start(new)
                else:
                    with InferenceProfiler.timer("beam_search.step"):
                        self._advance(live)
                for w in [w for w in live if w.group.done]:
                    for rid in w.rids:
                        if rid in self.mgr:
                            self.mgr.close(rid)
                    live.remove(w)
                    del held[w.index]
                    out[w.index] = BeamResponse(w.group.finished, len(w.prompt), (time.perf_counter() - w.t_start) * 1e3)
        finally:
            for w in live:                                 # (only when a step failed)
                for rid in w.rids:
                    if rid in self.mgr:
                        self.mgr.close(rid)
        return out

    def _room(self, need: int, held: Dict[int, int], n_live: int) -> bool:
        B = self.params.num_beams
        if (n_live + 1) * B > self.engine_config.max_num_seqs or (self.mgr.n_state_slots and (n_live + 1) * B > self.mgr.n_state_slots):
            return False
        return all(sum(held.values()) + need <= pool.n_pages for pool in self.mgr.pools)

    def _start(self, new: List[_Live]) -> None:
        """The prompts' portions, the first choice, and the beams that continue it."""
        cfg = self.engine_config
        done = [0] * len(new)
        for w in new:
            self.cache.reset_state(self.mgr.open(w.rids[0]))
        while any(d < len(w.prompt) for d, w in zip(done, new)):
            budget, entries, last = cfg.max_batch_tokens, [], []
            for k, w in enumerate(new):
                n = min(len(w.prompt) - done[k], cfg.max_chunk, budget)
                if n <= 0:
                    continue
                ends = done[k] + n == len(w.prompt)
                entries.append(StepEntry(w.rids[0], w.prompt[done[k]:done[k] + n], [n - 1] if ends else []))
                done[k] += n
                budget -= n
                if ends:
                    last.append(w)
            logits, ctx = self.runner.run(entries)
            if last:
                self._first_choice(last, logits)
        for w in new:
            if w.group.done:
                continue
            for rid in w.rids[1:]:
                self.mgr.fork(w.rids[0], rid)
        self._reorder([w for w in new if not w.group.done], [[0] * self.params.num_beams] * len(new))

    def _first_choice(self, group: List[_Live], logits: torch.Tensor) -> None:
        """Among one row of logits a prompt.  (The rows go in one by one as groups of one beam.)"""
        n, dev = len(group), logits.device
        chosen = torch.empty(4, n, self.n_keep, dtype=torch.int32, device=dev)
        ws = torch.empty(ops.beam_select_floats(n, 1, logits.shape[1]), device=dev)
        ops.beam_select(logits, torch.zeros(n, device=dev), 1, chosen[0].view(torch.float32), chosen[1], chosen[2], ws,
                        out_scores_low=chosen[3].view(torch.float32))
        for w, c in zip(group, self._candidates(chosen)):
            w.group.take(c)

    @staticmethod
    def _candidates(chosen: torch.Tensor) -> List[List[Tuple[float, int, int]]]:
        """(score, parent, token) of every place; a score is the sum of its two 32-bit parts."""
        scores, parents, tokens, low = chosen.cpu().numpy()
        scores = scores.view(np.float32).astype(np.float64) + low.view(np.float32)
        return [list(zip(s, p, t)) for s, p, t in zip(scores.tolist(), parents.tolist(), tokens.tolist())]

    def _advance(self, live: List[_Live]) -> None:
        """One token of every beam of every prompt, and the next choice."""
        B = self.params.num_beams
        entries, scores = [], []
        for w in live:
            for rid, tokens, score in zip(w.rids, w.group.tokens, w.group.scores):
                self.mgr.extend(rid, 1)
                entries.append(StepEntry(rid, [tokens[-1]], [0]))
                scores.append(score)
        shared = [[self._shared(w, g) for w in live] for g in range(len(self.cache.groups))]
        _, ctx = self.runner.run(entries, reserved=True, beams=BeamStep(B, self.n_keep, scores, shared))
        chosen = self._candidates(ctx.chosen)              # (waits for the step)
        for e in entries:
            self.mgr.commit(e.rid)
        parents = [w.group.take(c) for w, c in zip(live, chosen)]
        self._reorder([w for w in live if not w.group.done], [p for w, p in zip(live, parents) if not w.group.done])

    def _shared(self, w: _Live, group: int) -> int:
        """Positions in the pages with which all tables of the prompt's beams begin.  (What beams have in common stays common: they
        continue one of them.)"""
        tables = [self.mgr.table(rid, group) for rid in w.rids]
        n = w.shared_pages[group]
        while n < len(tables[0]) and all(t[n] == tables[0][n] for t in tables):
            n += 1
        w.shared_pages[group] = n
        return n * self.mgr.page_size

    def _reorder(self, live: List[_Live], parents: List[List[int]]) -> None:
        """Beam b of every prompt continues what beam parents[b] was: full pages by the tables, the rest on the device."""
        B = self.params.num_beams
        if not live or all(p == list(range(B)) for p in parents):
            return
        n = len(live)
        slots = [[self.mgr.state_slot(rid) for rid in w.rids] for w in live]
        writing = [[[self.mgr.writing(rid, g) for rid in w.rids] for w in live] for g in range(len(self.cache.groups))]
        for w, p in zip(live, parents):
            self.mgr.reorder(w.rids, p)
        words = torch.tensor([parents[:n], slots, *writing], dtype=torch.int32).to(self.runner.device)
        if self.cache.state:
            ops.state_reorder(list(self.cache.state.values()), words[1], words[0])
        for g, t in enumerate(self.cache._group_tensors):
            if any(p >= 0 for row in writing[g] for p in row):
                ops.state_reorder([t], words[2 + g], words[0], dim=1)
