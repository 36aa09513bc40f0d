"""The step function: one batch of (request, its next tokens) through the model.

A step may mix portions of prompts with single decoded tokens, cut anywhere.  It runs only
the tokens it is given, against the cache that earlier steps left, and returns the logits at
the wanted places.  The reference has two entry points for one request at a time
(``batchForward`` for a prompt in chunks of 512 and ``forward`` for one token:
core/src/main/java/io/teknek/deliverance/model/AbstractModel.java:1011-1048,1064-1072); both
collapse into this one function, and so does the head that its sampler applies to the last
row (core/.../model/AbstractGeneratorSampler.java:112-115).
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Hashable, List, Optional, Sequence

import numpy as np
import torch

from ..cache.manager import OutOfPages
from ..models.causal_lm import CausalLM
from ..parts.base import Arena, StepContext
from ..sampling.sampler import RECORD_WORDS
from .device_cache import DeviceCache


@dataclass
class StepEntry:
    rid: Hashable
    tokens: Sequence[int]
    want: Sequence[int] = field(default_factory=list)    # places among ``tokens`` whose logits are wanted
    # The entry's one token is not known on the host yet: it is row ``from_sampled`` of the tokens
    # that the step before sampled on the device (``StepRunner.sampled``); ``tokens`` holds a placeholder.
    from_sampled: Optional[int] = None


@dataclass
class BeamStep:
    """What a step of beam search brings beside its entries, which are the beams of one request after another, one token each."""
    n_beams: int                    # beams of a request
    n_keep: int                     # candidates that are wanted of every request
    scores: Sequence[float]         # the beams' summed log-probabilities, one an entry (-inf: no beam)
    shared: Sequence[Sequence[int]]  # per cache group and request: positions in pages that all its beams have in common


class StepError(ValueError):
    pass


class StepPacker:
    """The host side of a step: where each array of the step lies in its one buffer of integers,
    and the values that go there.  It reads the cache manager only, so it runs without a GPU."""

    def __init__(self, manager, n_groups: int, page_size: int):
        self.manager = manager
        self.n_groups = n_groups
        self.page_size = page_size

    def layout(self, entries, order, pad_to, max_blocks, extra, extra_a_pad=RECORD_WORDS):
        """Where each array of the step lies in its one buffer of integers: tokens, where a token
        comes from, positions, sequence ids, row starts, lengths, state slots, wanted rows, then
        per cache group the cache row of every token and the block tables, then ``extra`` (and
        ``extra_a_pad`` zeros for each sequence that is filled up).  With ``pad_to`` the step is filled up with
        empty one-token sequences (length 0, no cache row), so that its shape is fixed."""
        mgr = self.manager
        S_real = len(entries)
        n_pad = 0 if pad_to is None else pad_to - S_real
        N = sum(len(e.tokens) for e in entries) + n_pad
        S = S_real + n_pad
        R = sum(len(e.want) for e in entries) + n_pad
        G = self.n_groups
        if max_blocks is None:
            max_blocks = max(1, max(len(mgr.table(e.rid, g)) for e in entries for g in range(G))) if G else 1
        n_extra = 0 if not extra else len(extra) + extra_a_pad * n_pad
        offs = {}
        o = 0
        for name, n in (("tokens", N), ("token_src", N), ("positions", N), ("seq_of", N), ("q_start", S + 1),
                        ("seq_lens", S), ("state_slots", S), ("want", R)):
            offs[name] = (o, n)
            o += n
        for g in range(G):
            offs[f"slot_map{g}"] = (o, N)
            offs[f"block_table{g}"] = (o + N, S * max_blocks)
            o += N + S * max_blocks
        if n_extra:
            offs["extra"] = (o, n_extra)
            o += n_extra
        meta = dict(N=N, S=S, R=R, G=G, max_blocks=max_blocks, n_pad=n_pad,
                    n_decode=sum(1 for e in entries if len(e.tokens) == 1) + n_pad)
        return offs, meta, o

    def fill(self, buf, offs, meta, entries, order, starts, extra):
        """Write the step's integers into ``buf`` (a numpy view of pinned memory).  Long portions
        are written as arrays, single tokens as scalars."""
        mgr = self.manager
        ps = self.page_size

        def view(name):
            a, n = offs[name]
            return buf[a:a + n]
        tok, src, pos, seq = view("tokens"), view("token_src"), view("positions"), view("seq_of")
        q_start_v, seq_lens_v, state_v, want_v = view("q_start"), view("seq_lens"), view("state_slots"), view("want")
        G, mb, n_pad = meta["G"], meta["max_blocks"], meta["n_pad"]
        sms = [view(f"slot_map{g}") for g in range(G)]
        bts = [view(f"block_table{g}") for g in range(G)]
        for bt in bts:
            bt[:] = -1
        q_start, seq_lens, state_slots = [0], [], []
        row0 = {}
        row = 0
        for s, i in enumerate(order):
            e = entries[i]
            n = len(e.tokens)
            st = starts[e.rid]
            row0[i] = row
            if n == 1:
                tok[row] = e.tokens[0]
                src[row] = -1 if e.from_sampled is None else e.from_sampled
                pos[row] = st
                seq[row] = s
            else:
                tok[row:row + n] = e.tokens
                src[row:row + n] = -1
                pos[row:row + n] = np.arange(st, st + n, dtype=np.int32)
                seq[row:row + n] = s
            for g in range(G):
                t = mgr.table(e.rid, g)
                if n == 1:
                    page = t[st // ps]
                    if page < 0:
                        raise StepError(f"position {st} of {e.rid!r} lies in a page that was given back")
                    sms[g][row] = page * ps + st % ps
                else:
                    sms[g][row:row + n] = mgr.slots_for(e.rid, g, st, n)
                bts[g][s * mb:s * mb + len(t)] = t
            row += n
            q_start.append(row)
            seq_lens.append(st + n)
            state_slots.append(mgr.state_slot(e.rid))
        S_real = len(entries)
        r = 0
        for i, e in enumerate(entries):
            for w in e.want:
                want_v[r] = row0[i] + int(w)
                r += 1
        for k in range(n_pad):          # empty one-token sequences
            tok[row] = 0; src[row] = -1; pos[row] = 0; seq[row] = S_real + k
            for g in range(G):
                sms[g][row] = -1
            want_v[r] = row
            r += 1
            row += 1
            q_start.append(row); seq_lens.append(0); state_slots.append(-1)
        q_start_v[:] = q_start
        seq_lens_v[:] = seq_lens
        state_v[:] = state_slots
        if "extra" in offs:
            ex = view("extra")
            ex[:len(extra)] = extra
            ex[len(extra):] = 0
        meta.update(q_start=q_start, seq_lens=seq_lens, state_slots=state_slots)


class StepRunner:
    def __init__(self, model: CausalLM, cache: DeviceCache, use_graphs: bool = False, max_graph_batch: int = 256,
                 kernels: str = "tuned", native_step: bool = True):
        self.model = model
        self.cache = cache
        self.kernels = kernels                       # "tuned" | "reference" (EngineConfig.kernels)
        # the layer loop in one call into the library, where the model's parts allow it (engine/native_step.py)
        from .native_step import NativeStep
        self.joins_shares = NativeStep.takes(model, cache, kernels)
        self.native = NativeStep(model, cache) if native_step and self.joins_shares else None
        # (cache group, heads, key heads, head size, window) of the layers whose beams' shared pages can be read once
        self._beam_layers: Optional[List[tuple]] = None
        self._beam_choices = {}                      # what was estimated for steps of one shape and context (see _beams_attend)
        # hook(layer, stage, tensor) for named intermediates of every step; steps then run kernel by
        # kernel, never from a recorded graph
        self.debug_hook = None
        self.device = model.device
        self.arena = Arena(self.device)
        self.packer = StepPacker(cache.manager, len(cache.groups), cache.page_size)
        self._layout, self._fill = self.packer.layout, self.packer.fill
        self._staging: Optional[torch.Tensor] = None     # pinned host buffer for the step's integers
        self._staging_dev: Optional[torch.Tensor] = None
        self._copied = None
        # a request never holds more pages than the pool has, whatever the model's position limit
        self.max_blocks_cap = min(-(-model.config.max_positions // cache.page_size), max(1, cache.n_pages))
        self.last_ctx: Optional[StepContext] = None
        self.use_graphs = use_graphs and model.graph_safe
        self.max_graph_batch = max_graph_batch
        self._graphs = {}
        # where every sampling step leaves its tokens (row i: the i-th wanted row), and where a step
        # launched on top of it takes them from
        self.sampled = torch.zeros(2 * max(64, max_graph_batch), dtype=torch.int32, device=self.device)

    # ---- host -> device in one copy --------------------------------------------------------
    def _staging_for(self, n: int):
        """The pinned buffer (as a numpy view) that the step's ``n`` integers are written into."""
        if self._staging is None or self._staging.numel() < n:
            cap = max(4096, 2 * n)
            self._staging = torch.empty(cap, dtype=torch.int32, pin_memory=True)
            self._staging_np = self._staging.numpy()
            self._staging_dev = torch.empty(cap, dtype=torch.int32, device=self.device)
            self._copied = None
        if self._copied is not None:
            self._copied.synchronize()       # the last step's copy has read the pinned buffer
        return self._staging_np[:n]

    def _upload(self, n: int) -> torch.Tensor:
        self._staging_dev[:n].copy_(self._staging[:n], non_blocking=True)
        self._copied = torch.cuda.Event()
        self._copied.record()
        return self._staging_dev

    # ---- the step --------------------------------------------------------------------------
    def run(self, entries: Sequence[StepEntry], reserved: bool = False,
            sample_records: Optional[List[int]] = None, beams: Optional[BeamStep] = None):
        """Run one step.  Returns (logits [R, V] float32 on the device, ctx).  The rows follow
        the order of ``entries`` and of each entry's ``want``.  With ``reserved`` the caller has
        already opened the requests and reserved their positions (``CacheManager.extend``).
        ``sample_records`` (8 words per wanted row, see sampling.device_record) ride along in the
        same host-to-device copy (``ctx.extra``); when they are given and the step holds one-token
        sequences only, the step and its sampling are replayed from a recorded HIP graph and the
        sampled tokens are left in ``ctx.sampled`` (the first rows of ``self.sampled``).  With ``beams`` (in place of
        ``sample_records``) the step's entries are beams, one token each whose logits are wanted, and the choice of the next ones
        (``ops.beam_select``) is left in ``ctx.chosen``, int32 [4, requests, n_keep] on the device: the bits of the 32-bit scores, parents,
        tokens, and the bits of what the scores leave of the 64-bit sums."""
        mgr = self.cache.manager
        cfg = self.model.config
        if not entries:
            raise StepError("a step needs at least one entry")
        seen = set()
        for e in entries:
            if e.rid in seen:
                raise StepError(f"request {e.rid!r} appears twice in one step")
            seen.add(e.rid)
            if len(e.tokens) == 0:
                raise StepError(f"request {e.rid!r} brings no tokens")
            if len(e.tokens) <= 8:
                bad = [t for t in e.tokens if not (0 <= int(t) < cfg.vocab_size)]
            else:
                arr = np.asarray(e.tokens, dtype=np.int64)
                bad = arr[(arr < 0) | (arr >= cfg.vocab_size)].tolist()
            if bad:
                raise StepError(f"request {e.rid!r}: token id {bad[0]} is outside the vocabulary of {cfg.vocab_size}")
            for w in e.want:
                if not (0 <= int(w) < len(e.tokens)):
                    raise StepError(f"request {e.rid!r}: wanted place {w} is outside its {len(e.tokens)} tokens")
            if e.from_sampled is not None and not (len(e.tokens) == 1 and 0 <= e.from_sampled < self.sampled.numel()):
                raise StepError(f"request {e.rid!r}: only a single token can come from the sampled tokens")

        if beams is not None:
            if sample_records is not None or any(len(e.tokens) != 1 or list(e.want) != [0] for e in entries):
                raise StepError("beams bring one token each, whose logits are wanted, and no sampling records")
            n = len(entries) // max(1, beams.n_beams)
            if n * beams.n_beams != len(entries) or len(beams.scores) != len(entries) or \
                    [len(p) for p in beams.shared] != [n] * len(self.cache.groups):
                raise StepError(f"{len(entries)} entries, {len(beams.scores)} scores, groups of {beams.n_beams} beams")

        starts = {}
        opened = []
        if reserved:
            for e in entries:               # the entry's tokens are the last positions that were reserved
                starts[e.rid] = mgr.length(e.rid) + mgr.pending(e.rid) - len(e.tokens)
                if starts[e.rid] < mgr.length(e.rid):
                    raise StepError(f"request {e.rid!r} brings {len(e.tokens)} tokens, {mgr.pending(e.rid)} are reserved")
        else:
            done = []
            try:
                for e in entries:
                    if e.rid not in mgr:
                        self.cache.reset_state(mgr.open(e.rid))
                        opened.append(e.rid)
                    if mgr.length(e.rid) + len(e.tokens) > cfg.max_positions:
                        raise StepError(f"request {e.rid!r} would reach position "
                                        f"{mgr.length(e.rid) + len(e.tokens)}, the model has {cfg.max_positions}")
                    starts[e.rid] = mgr.extend(e.rid, len(e.tokens))
                    done.append(e.rid)
            except (OutOfPages, StepError):
                for rid in done:
                    mgr.rollback(rid)
                for rid in opened:
                    mgr.close(rid)
                raise

        # one-token entries first (the decode kernels take them), portions after
        order = sorted(range(len(entries)), key=lambda i: (len(entries[i].tokens) != 1, i))
        n_decode = sum(1 for e in entries if len(e.tokens) == 1)
        from ..profiler import KernelProfiler
        graph_ok = ((sample_records is not None or beams is not None) and n_decode == len(entries) and self.use_graphs
                    and self.debug_hook is None and not KernelProfiler.enabled
                    and len(entries) <= self.max_graph_batch and all(list(e.want) == [0] for e in entries))
        from ..kernels import ops
        try:
            with ops.kernel_mode_scope(self.kernels):
                if graph_ok:
                    logits, ctx = self._run_graph(entries, starts, sample_records, beams)
                else:
                    logits, ctx = self._run_eager(entries, order, starts, sample_records, beams)
        except Exception:
            # A launch that was refused (a size no kernel takes) leaves nothing half-done on the host:
            # what this call reserved goes back, requests it opened are closed.  A caller that
            # reserved itself decides what becomes of its requests.
            if not reserved:
                for e in entries:
                    mgr.rollback(e.rid)
                for rid in opened:
                    mgr.close(rid)
            raise
        if not reserved:                 # who reserves commits: the scheduler does it for its batches
            for e in entries:
                mgr.commit(e.rid)
        return logits, ctx

    @staticmethod
    def _beam_words(beams: BeamStep, n_requests: int) -> List[int]:
        """The beams' scores (as the bits of 32-bit floats) and, per cache group, the shared positions, for ``n_requests``
        requests, of which those behind the step's own are empty."""
        n = n_requests * beams.n_beams
        scores = np.full(n, -np.inf, dtype=np.float32)
        scores[:len(beams.scores)] = beams.scores
        words = scores.view(np.int32).tolist()
        for per_request in beams.shared:
            words += list(per_request) + [0] * (n_requests - len(per_request))
        return words

    @staticmethod
    def _beam_low_words(beams: BeamStep, n_requests: int) -> List[int]:
        """What the 32-bit scores of ``_beam_words`` leave of the beams' scores, as the bits of 32-bit floats."""
        scores = np.asarray(beams.scores, dtype=np.float64)
        near = scores.astype(np.float32)
        low = np.zeros(n_requests * beams.n_beams, dtype=np.float32)
        np.subtract(scores, near, out=low[:len(scores)], where=np.isfinite(near), casting="same_kind")
        return low.view(np.int32).tolist()

    def _take_beams(self, ctx, beams: BeamStep) -> None:
        """Where the step's arrays of beam search lie in ``ctx.extra``."""
        n, G = ctx.n_seqs, len(self.cache.groups)
        per = n // beams.n_beams
        ctx.n_beams = beams.n_beams
        ctx.beam_scores = ctx.extra[:n].view(torch.float32)
        ctx.beam_shared_host = beams.shared
        ctx.beam_shared = [ctx.extra[n + g * per:n + (g + 1) * per] for g in range(G)]
        ctx.beam_scores_low = ctx.extra[n + G * per:2 * n + G * per].view(torch.float32)

    def _choose(self, ctx, beams: BeamStep, logits: torch.Tensor):
        from ..kernels import ops
        per = ctx.n_seqs // beams.n_beams
        chosen = ctx.flat("beam_chosen", 4 * per * beams.n_keep, torch.int32).view(4, per, beams.n_keep)
        ws = ctx.flat("beam_select", ops.beam_select_floats(logits.shape[0], beams.n_beams, logits.shape[1]), torch.float32)
        ops.beam_select(logits, ctx.beam_scores, beams.n_beams, chosen[0].view(torch.float32), chosen[1], chosen[2], ws,
                        ctx.beam_scores_low, chosen[3].view(torch.float32))
        return chosen

    def _run_eager(self, entries, order, starts, sample_records, beams=None):
        from ..kernels import ops
        extra = sample_records
        if beams is not None:
            n = len(entries) // beams.n_beams
            extra = self._beam_words(beams, n) + self._beam_low_words(beams, n)
        offs, meta, n_words = self._layout(entries, order, pad_to=None, max_blocks=None, extra=extra)
        self._fill(self._staging_for(n_words), offs, meta, entries, order, starts, extra)
        dev = self._upload(n_words)
        ctx = self._context(dev, offs, meta, self.arena)
        if beams is not None:
            self._take_beams(ctx, beams)
            ctx.beams_attend = self._beams_attend(beams, [starts[e.rid] + 1 for e in entries[::beams.n_beams]], meta["S"], meta["max_blocks"], recorded=False)
        ctx.debug_hook = self.debug_hook
        self.last_ctx = ctx
        R = meta["R"]
        if any(e.from_sampled is not None for e in entries):
            ops.take_tokens(ctx.tokens, ctx.token_src, self.sampled, self.model.config.vocab_size)
        logits = self._forward(ctx, ctx.want_rows if R else None, R)
        if beams is not None:
            ctx.chosen = self._choose(ctx, beams, logits)
        return logits, ctx

    def _forward(self, ctx, want_rows, n_want):
        """The model's forward pass of this step: from C++ in one call, or part by part (always with the
        debug hook or the kernel profiler, which look between the kernels)."""
        from ..profiler import KernelProfiler
        if self.native is not None and ctx.debug_hook is None and not KernelProfiler.enabled and not ctx.beams_attend:
            return self.native.forward(ctx, want_rows, n_want)
        return self.model.forward(ctx, want_rows, n_want)

    # us that a layer of a step that is not recorded takes the host when it is issued part by part in place of one call into the library
    # (12 layers, a step of 4 or 64 rows: 0.45 and 1.00 ms, 1.23 and 1.76)
    PART_BY_PART_US = 46.0

    def _beams_attend(self, beams: BeamStep, lens: Sequence[int], n_seqs: int, max_blocks: int, recorded: bool) -> frozenset:
        """The layers (``StepContext.beams_attend``) of a step of ``n_seqs`` sequences in tables of ``max_blocks`` pages whose attention reads
        what beams share once, by what its requests (of ``lens`` positions) see and share.  (The calls that are issued from C++ do not
        know of it: a step that is not recorded leaves them only for more than that costs the host.)"""
        from ..kernels import ops
        from ..profiler import KernelProfiler
        if beams.n_beams < 2:
            return frozenset()
        if self._beam_layers is None:
            found = [(self.cache.group_of_slot[c.cache + k], *rest) for c in self.model.config.schedule
                     for k, *rest in getattr(self.model.blocks[c.layer].mixer, "paged_attention", tuple)()]
            self._beam_layers = sorted(set(found))
        native = self.native is not None and not recorded and self.debug_hook is None and not KernelProfiler.enabled
        n, seen = len(lens), []
        for group, _, _, _, window in self._beam_layers:
            shared = beams.shared[group]
            if window:
                gone = [max(0, m - window) for m in lens]
                seen.append((sum(min(m, window) for m in lens) // n, sum(max(0, s - g) for s, g in zip(shared, gone)) // n))
            else:
                seen.append((sum(lens) // n, sum(shared) // n))
        # (estimated once for contexts that are alike, of the next 16 positions: an estimate takes the host 12 us)
        key = (n_seqs, beams.n_beams, max_blocks, native, tuple((v // 16, s // 16) for v, s in seen))
        attend = self._beam_choices.get(key)
        if attend is None:
            attend = frozenset(layer for layer, (v, s) in zip(self._beam_layers, key[4]) if ops.attention_beams_pays(
                n_seqs // beams.n_beams, beams.n_beams, *layer[1:4], self.cache.page_size, max_blocks, self.model.dtype, 16 * v + 15, 16 * s,
                host_us=self.PART_BY_PART_US if native else 0.0))
            if len(self._beam_choices) >= 4096:
                self._beam_choices.clear()
            self._beam_choices[key] = attend
        return attend

    def _context(self, dev, offs, meta, arena) -> StepContext:
        def view(name):
            a, n = offs[name]
            return dev[a:a + n]
        N, S, G, max_blocks = meta["N"], meta["S"], meta["G"], meta["max_blocks"]
        ctx = StepContext()
        ctx.device = self.device
        ctx.dtype = self.model.dtype
        ctx.joins_shares = self.joins_shares
        ctx.n_tokens, ctx.n_seqs, ctx.n_decode = N, S, meta["n_decode"]
        ctx.tokens, ctx.positions, ctx.seq_of_token = view("tokens"), view("positions"), view("seq_of")
        ctx.token_src = view("token_src")
        ctx.q_start, ctx.seq_lens, ctx.state_slots = view("q_start"), view("seq_lens"), view("state_slots")
        ctx.q_start_host, ctx.seq_lens_host, ctx.state_slots_host = meta["q_start"], meta["seq_lens"], meta["state_slots"]
        ctx.max_query_len = max(meta["q_start"][s + 1] - meta["q_start"][s] for s in range(S))
        ctx.max_seq_len = max(meta["seq_lens"])
        ctx.block_tables = [view(f"block_table{g}").view(S, max_blocks) for g in range(G)]
        ctx.slot_maps = [view(f"slot_map{g}") for g in range(G)]
        ctx.cache = self.cache
        ctx._arena = arena
        ctx.extra = view("extra") if "extra" in offs else None
        ctx.want_rows = view("want")
        return ctx

    # ---- decode-only steps replayed from a HIP graph ----------------------------------------------
    # Recordings of beam search's steps that are kept, with their scratch buffers: those that were used last.  (A search whose prompts end one after another
    # and that goes over to the other attention has two for each power of two of requests.)
    MAX_BEAM_RECORDINGS = 16

    @staticmethod
    def _bucket(n: int) -> int:
        return 1 << (n - 1).bit_length()

    def _beam_bucket(self, n_seqs: int, n_beams: int) -> int:
        """Beams are padded request by request, to no more of them than the engine takes."""
        return min(self._bucket(n_seqs // n_beams), max(n_seqs, self.max_graph_batch) // n_beams) * n_beams

    def _keep_recording(self, key) -> None:
        """The recording (or the one that is about to be made) was used last; the one that was not for the longest time goes."""
        if key in self._graphs:
            self._graphs[key] = self._graphs.pop(key)
            return
        of_beams = [k for k in self._graphs if isinstance(k, tuple)]
        if len(of_beams) >= self.MAX_BEAM_RECORDINGS:
            torch.cuda.synchronize()                       # (its last replay may be under way)
            del self._graphs[of_beams[0]]

    def _run_graph(self, entries, starts, sample_records, beams=None):
        """A step of one-token sequences only has a fixed shape once it is padded to a bucket
        size, so its kernels (model and sampling, or the choice among beams) are recorded once per bucket and
        replayed.  Only the step's integers change: they are copied into the bucket's own buffer first."""
        from ..kernels import ops
        S = len(entries)
        bucket = self._bucket(S) if beams is None else self._beam_bucket(S, beams.n_beams)
        order = list(range(S))
        extra, a_pad = sample_records, RECORD_WORDS
        if beams is not None:
            n = bucket // beams.n_beams
            extra, a_pad = self._beam_words(beams, n) + self._beam_low_words(beams, n), 0
        offs, meta, n_words = self._layout(entries, order, pad_to=bucket, max_blocks=self.max_blocks_cap, extra=extra, extra_a_pad=a_pad)
        key, attend = bucket, None
        if beams is not None:                              # (a step's kernels are recorded: which attention they hold is part of its name)
            attend = self._beams_attend(beams, [starts[e.rid] + 1 for e in entries[::beams.n_beams]], bucket, self.max_blocks_cap, recorded=True)
            key = (bucket, beams.n_beams, beams.n_keep, attend)
        st = self._graphs.get(key)
        if beams is not None:
            self._keep_recording(key)
        if st is None:
            host = torch.empty(n_words, dtype=torch.int32, pin_memory=True)
            st = {"dev": torch.empty(n_words, dtype=torch.int32, device=self.device),
                  "host": host, "host_np": host.numpy(),
                  "arena": Arena(self.device), "graph": None, "copied": None}
            self._graphs[key] = st
        assert st["dev"].numel() == n_words, "a bucket's layout is fixed"
        if st["copied"] is not None:
            st["copied"].synchronize()
        self._fill(st["host_np"], offs, meta, entries, order, starts, extra)
        st["dev"].copy_(st["host"], non_blocking=True)
        st["copied"] = torch.cuda.Event()
        st["copied"].record()
        ctx = self._context(st["dev"], offs, meta, st["arena"])
        self.last_ctx = ctx
        if beams is not None:
            ctx.beams_attend = attend
            if st["graph"] is None:                        # (a recorded step knows where they lie)
                self._take_beams(ctx, beams)

        sampled = self.sampled[:bucket]

        def body():
            ops.take_tokens(ctx.tokens, ctx.token_src, self.sampled, self.model.config.vocab_size)
            logits = self._forward(ctx, ctx.want_rows, bucket)
            if beams is None:
                ops.sample(logits, ctx.extra, sampled)
            else:
                st["chosen"] = self._choose(ctx, beams, logits)
            return logits

        if st["graph"] is None:
            st["logits"] = body()                      # eager once: sizes the bucket's scratch buffers
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                st["logits"] = body()
            st["graph"] = g
            # the eager run above already did this step's work; the recorded graph is used from the next step on
        else:
            st["graph"].replay()
        if beams is None:
            ctx.sampled = sampled[:S]
        else:
            ctx.chosen = st["chosen"][:, :S // beams.n_beams]
        return st["logits"][:S], ctx
