"""Several continuations of every prompt, decoded together over ONE copy of the prompt's cache.

:func:`sample_many` runs each prompt once.  Its continuations share the prompt's whole pages (``csrc/attn_shared.cuh``: a step reads them
once for all continuations, short ones once per eight rows); the rest of the prompt's last page is copied, and per-sequence records are, so that what a
continuation writes is its own.  From then on a step needs nothing from the host: the page tables grow on the device, out of a list of
pages lent to the batch (``ops.step_tables``), the rules are applied and the token is drawn there, and the host, one step behind, reads the
ids.  A step's description is uploaded only when a continuation has ended, or another batch has decoded by the same captured step.

Attention is cut by the lengths of the whole batch: in its last places a continuation's logits depend on what is decoded beside it.

Models whose attention is not over paged keys and values, or has options that the shared form does not take, decode the same way: their
mixers read the page tables, in which the shared pages stand like any others.
"""
from __future__ import annotations

import collections
import dataclasses
import time
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from .. import ops
from ..layout import PAGE, pages_for
from ..sampling.rules import LogitRules, Steering
from ..sampling.sampler import rng_state
from .generate import GenOptions, GenResult, stop_set
from .run import DeviceRun


def _power(n: int, least: int = 1) -> int:
    p = least
    while p < n:
        p *= 2
    return p


def pages_of_batch(prompt: int, limit: int, n: int) -> int:
    """Pages that a prompt of ``prompt`` tokens and ``n`` continuations of up to ``limit`` take: the prompt's, and behind its whole ones each
    continuation's own, and one more (a continuation that has ended rides along for one step, which may open a page)."""
    return pages_for(prompt) + n * (pages_for(prompt % PAGE + limit) + 1)


class SampleRun(DeviceRun):
    """The batch of :func:`sample_many`: ``start`` runs the prompts and forks them, ``launch`` and ``collect`` are as in
    :class:`~wick_b200.engine.run.DeviceRun`.  A continuation is named by its number among all of the batch."""

    def __init__(self, engine, cfg, stop_token_ids=(), rules: Optional[Sequence[Optional[LogitRules]]] = None):
        super().__init__(engine, cfg, stop_token_ids, None)
        self.rules_of_prompt = rules
        self.lent: List[int] = []
        self.slots: List[int] = []
        self.parents: List[int] = []
        self.mark = object()         # of this batch, on the captured step that holds its description

    def start(self, prompts: Sequence[Sequence[int]], numbers: Sequence[Sequence[int]], limits: Sequence[int]) -> None:      # type: ignore[override]
        """numbers[i]: which continuations of prompt i (their generators are seeded by them); limits[i]: the tokens each may have."""
        e, cache, dev = self.engine, self.engine.cache, self.engine.device
        P = len(prompts)
        lens, whole = [len(p) for p in prompts], [len(p) // PAGE for p in prompts]
        self.whole = whole
        self.prompt_of = [i for i in range(P) for _ in numbers[i]]
        R = len(self.prompt_of)
        self.prompt_len = [lens[i] for i in self.prompt_of]
        self.length = list(self.prompt_len)                        # positions cached, of each continuation
        self.limit = [limits[i] for i in self.prompt_of]
        # the prompts, once each
        self.parents = [e.open_seq() for _ in prompts]
        for s, p in zip(self.parents, prompts):
            cache.reserve(s, len(p))
        logits, _ = e._forward_prompt(self.parents, [list(p) for p in prompts], [[n - 1] for n in lens], [0] * P, lens)
        for s, n in zip(self.parents, lens):
            cache.advance(s, n)
        # the continuations' places
        self.slots = [e.open_seq() for _ in range(R)]
        self.lent = cache.lend(sum(pages_of_batch(n, lim, len(k)) - pages_for(n) for n, lim, k in zip(lens, limits, numbers)))
        self.width = _power(max(pages_for(n + lim) + 1 for n, lim in zip(lens, limits)), 8)
        self.own_bound = _power(max(n - w * PAGE + lim + 1 for n, w, lim in zip(lens, whole, limits)), PAGE)
        tables = np.zeros((cache.max_seqs + 1, self.width), dtype=np.int32)
        for s in self.parents:
            tables[s, :len(cache.pages_of(s))] = cache.pages_of(s)
        up = lambda v: torch.from_numpy(np.ascontiguousarray(v, dtype=np.int32)).pin_memory().to(dev, non_blocking=True)     # noqa: E731
        self.tables, self.free = up(tables), up(self.lent)
        self.heads = torch.zeros((2, 1), dtype=torch.int32, device=dev)
        self.head = 0
        # fork: whole pages by name, a page of the list for what lies behind them, the tail's contents copied into it
        tail = [lens[i] - whole[i] * PAGE for i in self.prompt_of]
        slots = up(self.slots)
        make = lambda n, t=torch.int32: torch.empty(n, dtype=t, device=dev)      # noqa: E731
        fork = dict(page_table=make((R, self.width)), cu_seqlens=make(R + 1), kv_len=make(R), positions=make(sum(tail)), seq_of_token=make(sum(tail)),
                    slot_map=make(sum(tail), torch.int64))
        ops.step_tables(up([whole[i] * PAGE for i in self.prompt_of]), up(tail), slots, self.tables, self.free, self.heads[0], head_out=self.heads[1],
                        parent=up([self.parents[i] for i in self.prompt_of]), **fork)
        self.head = 1
        cut = [r for r in range(R) if tail[r]]
        if cut:
            src = up([cache.pages_of(self.parents[self.prompt_of[r]])[whole[self.prompt_of[r]]] for r in cut]).long()
            dst = fork["page_table"][up(cut).long(), up([whole[self.prompt_of[r]] for r in cut]).long()].long()
            cache.copy_pages(src, dst)
        cache.copy_slots(up([self.parents[i] for i in self.prompt_of]).long(), slots.long())
        # sampling state: a generator and a history for each
        self._buffers(R)
        if self.cfg.temperature > 0.0:
            self.rng = torch.tensor([rng_state(self.cfg.seed + k) for ks in numbers for k in ks], dtype=torch.int64).to(dev)
        rows = torch.arange(R, dtype=torch.int32, device=dev)
        rules = [None] * P if self.rules_of_prompt is None else list(self.rules_of_prompt)
        if Steering.wanted(rules) or self.cfg.repetition_penalty != 1.0:
            self.steering = Steering([rules[i] or LogitRules() for i in self.prompt_of], self.cfg.repetition_penalty, self.vocab, dev)
            told = up([t for i in self.prompt_of for t in prompts[i]])
            self.steering.said(told, rows.repeat_interleave(up([lens[i] for i in self.prompt_of])), generated=False)
        rec = np.zeros((R, ops.SEQ_STATE_WORDS), dtype=np.int32)
        rec[:, ops.SEQ_LIMIT], rec[:, ops.SEQ_ROW] = self.limit, np.arange(R)
        ops.seq_state_set(e.seq_state, slots, up(rec))
        self.graph = None
        first = logits[:P].repeat_interleave(up([len(k) for k in numbers]), 0)
        with ops.stream_scope():
            self._sample_and_advance(first, slots, up(self.length), R, rows)
        self.last_logits = first

    def launch(self, live: Sequence[int]) -> None:                   # type: ignore[override]
        e = self.engine
        B = len(live)
        # (The step is the engine's: another batch may have written its own description there since.)
        if self.graph is None or self.graph.composition != (self.mark, tuple(live)):
            self._compose(live)
        g, b = self.graph, self.graph.batch
        with ops.stream_scope():
            ops.step_prepare(e.seq_state, b.slots, b.tokens, b.positions, b.start, b.kv_len)
            ops.step_tables(b.start, g.ones, b.slots, self.tables, self.free, self.heads[self.head], page_table=b.page_table, cu_seqlens=b.cu_seqlens,
                            kv_len=b.kv_len, positions=b.positions, seq_of_token=b.seq_of_token, slot_map=g.slot_map, head_out=self.heads[1 - self.head])
            self.head = 1 - self.head
            if e.use_graphs:
                g.graph.replay()
                ops.launches[0] += g.kernels
                logits = g.logits
            else:
                b.memo.clear()
                logits = e.model.forward(b, e.cache)
            self._sample_and_advance(logits[:B], b.slots[:B], b.kv_len[:B], B, g.rows[:B])
        self.last_logits = logits[:B]
        for r in live:
            self.length[r] += 1

    def _compose(self, live: Sequence[int]) -> None:
        """The description of a step of these continuations; padded entries are a last group that shares nothing."""
        e, P, G = self.engine, len(self.parents), _power(len(self.parents) + 1)
        # (A batch that has shrunk and will end within 64 steps keeps the captured step it has.)
        ending = max(self.prompt_len[r] + self.limit[r] - self.length[r] for r in live) < 64
        g = self.graph = e.shared_graph(len(live), self.width, G, _power(max(self.whole)) if max(self.whole) else 0, self.own_bound, prefer_captured=ending)
        pad = g.n_pad - len(live)
        sizes = [0] * G
        for r in live:
            sizes[self.prompt_of[r]] += 1
        sizes[G - 1] = pad
        fields = [[self.slots[r] for r in live] + [0] * pad, np.cumsum([0] + sizes), self.whole + [0] * (G - P),
                  [self.prompt_of[r] for r in live] + [G - 1] * pad, list(live) + [-1] * pad]
        flat = torch.from_numpy(np.concatenate([np.asarray(f, dtype=np.int32) for f in fields])).pin_memory().to(e.device, non_blocking=True)
        at = 0
        for dst in (g.batch.slots, g.batch.shared.cu_groups, g.batch.shared.pages, g.batch.shared.group_of, g.rows):
            dst.copy_(flat[at:at + dst.numel()])
            at += dst.numel()
        self.uploads += 1
        self.h2d_bytes += flat.numel() * 4
        g.composition = (self.mark, tuple(live))

    def close(self) -> None:
        """Give back every slot and page."""
        for s in self.parents + self.slots:
            self.engine.close_seq(s)
        self.engine.cache.give_back(self.lent)
        self.parents, self.slots, self.lent = [], [], []


def sample_many(engine, prompts: Sequence[Sequence[int]], n: int, opts: Optional[GenOptions] = None,
                rules: Optional[Sequence[Optional[LogitRules]] | LogitRules] = None) -> List[List[GenResult]]:
    """``n`` continuations of every prompt, each prompt's in order.  Continuation k of a prompt draws with the generator of seed
    ``opts.sampler.seed + k``.  rules: for all prompts, or one for each (default: ``opts.rules``).  As many prompts as the batch limit
    (counted in continuations, 8,192 at the most), 1,023 of them, the cache's slots and its free pages allow are decoded together; a prompt with
    more continuations than the batch limit is run again for the rest of them.  A cache with a kind of storage that cannot be copied is refused."""
    opts = opts or GenOptions()
    if n < 1:
        raise ValueError(f"{n} continuations (at least 1)")
    rules = opts.rules if rules is None else rules
    per_prompt = [rules] * len(prompts) if rules is None or isinstance(rules, LogitRules) else list(rules)
    if len(per_prompt) != len(prompts):
        raise ValueError("one set of rules for all prompts, or one for each")
    stops = stop_set(engine, opts)
    cache = engine.cache
    if cache.cannot_copy():
        raise RuntimeError("the cache cannot be forked: storage of kind " + ", ".join(cache.cannot_copy()) + " does not say how its pages and records "
                           "are copied (Storage.copy_pages, Storage.copy_slots)")
    context = min(opts.context, cache.max_position or opts.context)
    most = min(opts.max_batch, ops.MAX_TABLE_SEQS)                  # continuations of a batch
    if most < 1:
        raise ValueError(f"a batch of {opts.max_batch} (at least 1)")
    results: List[List[Optional[GenResult]]] = [[None] * n for _ in prompts]
    waiting: List[Tuple[int, List[int], int]] = []                 # prompt, continuations, tokens each
    for i, p in enumerate(prompts):
        if len(p) == 0:
            raise ValueError("empty prompt")
        if len(p) > context:
            raise ValueError(f"prompt is {len(p)} tokens, context is {context}")
        limit = min(opts.max_tokens, context - len(p))
        if limit == 0:
            results[i] = [GenResult([], len(p), "length") for _ in range(n)]
            continue
        waiting += [(i, list(range(k, min(n, k + most))), limit) for k in range(0, n, most)]
    while waiting:
        chosen, rows, pages, slots = 0, 0, 0, 0
        for i, ks, limit in waiting[:ops.MAX_SHARED_GROUPS - 1]:     # (one group is the padding's)
            rows, slots, pages = rows + len(ks), slots + 1 + len(ks), pages + pages_of_batch(len(prompts[i]), limit, len(ks))
            if rows > most or slots > cache.slots.n_free or pages > cache.pages.n_free:
                break
            chosen += 1
        if chosen == 0:
            i, ks, limit = waiting[0]
            raise RuntimeError(f"{len(ks)} continuations of prompt {i} need {pages_of_batch(len(prompts[i]), limit, len(ks))} cache pages of {PAGE} tokens "
                               f"and {1 + len(ks)} slots; {cache.pages.n_free} pages and {cache.slots.n_free} slots are free")
        batch, waiting = waiting[:chosen], waiting[chosen:]
        run = SampleRun(engine, opts.sampler, stops, [per_prompt[i] for i, _, _ in batch])
        try:
            _decode(run, batch, prompts, stops, results)
        finally:
            run.close()
        engine.check_kernels()
    return results  # type: ignore[return-value]


@dataclasses.dataclass
class _Live:
    number: int                                                    # of the batch
    prompt: int
    k: int
    limit: int
    out: List[int] = dataclasses.field(default_factory=list)
    launched: int = 1
    done: bool = False


def _decode(run: SampleRun, batch, prompts, stops, results) -> None:
    live: List[_Live] = []
    for i, ks, limit in batch:
        live += [_Live(len(live) + j, i, k, limit) for j, k in enumerate(ks)]
    t0 = time.perf_counter()
    run.start([prompts[i] for i, _, _ in batch], [ks for _, ks, _ in batch], [limit for _, _, limit in batch])
    pending = collections.deque([list(live)])
    t1, prompt_ms = t0, 0.0
    while True:
        while len(pending) < run.depth + 1:
            rows = [s for s in live if not s.done and s.launched < s.limit]
            if not rows:
                break
            run.launch([s.number for s in rows])
            for s in rows:
                s.launched += 1
            pending.append(rows)
        if not pending:
            break
        rows = pending.popleft()
        toks = run.collect()
        now = time.perf_counter()
        if t1 == t0:
            t1, prompt_ms = now, (now - t0) * 1e3
        for s, tok in zip(rows, toks):
            if s.done:
                continue                                           # it rode along after its end
            finish = "stop" if int(tok) in stops else None
            if finish is None:
                s.out.append(int(tok))
                finish = "length" if len(s.out) >= s.limit else None
            if finish:
                s.done = True
                results[s.prompt][s.k] = GenResult(s.out, len(prompts[s.prompt]), finish, prompt_ms, (now - t1) * 1e3)
        live = [s for s in live if not s.done]
