"""Beam search over the paged cache, with nothing of a step decided on the host.

The reference decodes each sequence by sampling (serving/executor.py:334-393) and has no search.  Here a search's beams are
requests of the cache manager: the first holds the prompt, the others are its forks (`CacheManager.fork_request`), so the prompt's whole
pages lie in the cache once.  After the prompt's portions a step of all searches is one train of launches: the forward of every beam's
last token, the candidates (`ops.beam_candidates`), what of them goes on (`ops.beam_advance`), states and pages that follow
(`ops.beam_reorder`), and the next step's description (`ops.step_tables`).  What a step reads lies in one int32 buffer and what it makes for the next one in a
second one, which is then copied over the first: no operator writes what another still reads, and the copy stands between the kernels that make the block
tables and the attention kernels, which read them before they wait for the kernel before.  The train is captured as a CUDA graph; the host
replays it and copies each step's tokens and parents back behind it, one step late for the question whether all searches are over, and follows the parents
when they are.
"""

from __future__ import annotations

from collections import OrderedDict
from dataclasses import dataclass, replace

import numpy as np
import torch

from .. import ops
from ..cache.pools import OutOfPages
from ..sampling.params import BeamParams
from .batch import BatchLayout, context
from .engine import Engine, StepEntry
from .graphs import DecodeGraphs, captured


@dataclass
class BeamResult:
    ids: list                  # generated token ids (a stop id is not among them)
    score: float               # cumulative log-probability over n ** length_penalty
    finish_reason: str         # "stop" | "length"


class _Searches:
    """``G`` searches of ``params.beams`` beams whose contexts end within ``bucket`` tokens: the two buffers, the train of launches and its graph."""

    def __init__(self, engine: Engine, G: int, params: BeamParams, bucket: int):
        cache, self.G, self.params = engine.cache, G, params
        B, W = params.beams, params.results
        R = self.R = G * B
        columns = [cache.pages_for(bucket, gi) for gi in range(len(cache.groups))]
        # (tokens, parents, done in a row: what goes back to the host; parents are a step's own)
        extras = {"tokens": R, "parents": R, "done": G, "scores": R, "lengths": G, "pool_scores": G * W, "pool_lengths": G * W, "pool_parents": G * W, "pool_tokens": G * W}
        extras |= {f"pages{gi}": R * c for gi, c in enumerate(columns)}
        self.layout = layout = BatchLayout(R, R, R, columns, extras=extras)
        pin = engine.device.type == "cuda"
        self.host = torch.zeros(layout.total, dtype=torch.int32, pin_memory=pin)
        self.live = torch.zeros(layout.total, dtype=torch.int32, device=engine.device)
        self.next = torch.zeros_like(self.live)
        self.ones = torch.ones(R, dtype=torch.int32, device=engine.device)
        self.first = torch.zeros((G, B), dtype=torch.int32, device=engine.device)
        self.stop_ids = torch.tensor(params.stop_ids, dtype=torch.int32, device=engine.device) if params.stop_ids else None
        self.ctx = context(layout, self.live, cache.page_size, [1] * R, [bucket] * R, is_graph_replay=pin)
        self.ctx.token_ids = layout.sec(self.live, "tokens")
        self.page_size = cache.page_size
        self.strides = [g.need.stride for g in cache.groups]
        self.storage = list(cache.kv_storage)
        self.states = list(cache.state_storage.values())
        self.back = (layout.offs["tokens"], layout.offs["scores"])
        self.graph = None
        self.launches = self.reporting = 0
        # the places in both buffers, made once
        sec, f32 = layout.sec, torch.float32

        def places(buf):
            pool = ops.BeamPool(sec(buf, "pool_scores").view(f32).view(G, W), *(sec(buf, f"pool_{k}").view(G, W) for k in ("lengths", "parents", "tokens")))
            step = ops.BeamStep(sec(buf, "scores").view(f32).view(G, B), sec(buf, "parents").view(G, B), sec(buf, "tokens").view(G, B), sec(buf, "lengths"), sec(buf, "done"), pool)
            pages = [sec(buf, f"pages{gi}").view(R, c) for gi, c in enumerate(columns)]
            tables = ops.StepTables(sec(buf, "q_start"), sec(buf, "ctx_len"), sec(buf, "positions"), sec(buf, "seq_of_token"),
                                    tuple(sec(buf, f"block_tables{gi}").view(R, c) for gi, c in enumerate(columns)),
                                    tuple(sec(buf, f"slot_mapping{gi}") for gi in range(len(columns))))
            return step, sec(buf, "state_slots"), pages, tables
        self.now, self.then = places(self.live), places(self.next)

    def begin(self, engine: Engine, rows) -> None:
        """``rows``: the cache manager's requests, beam by beam."""
        h, sec, layout = self.host.numpy(), self.layout.sec, self.layout
        h[:] = 0
        for name in ("scores", "pool_scores"):
            sec(h, name).view(np.float32)[:] = -np.inf
        sec(h, "logit_rows")[:] = np.arange(self.R)
        for r, req in enumerate(rows):
            sec(h, "state_slots")[r] = req.slot
            sec(h, "ctx_len")[r] = req.num_tokens
            for gi, c in enumerate(layout.pages):
                own = sec(h, f"pages{gi}").reshape(self.R, c)[r]
                own[:] = -1
                own[:len(req.tables[gi])] = req.tables[gi]
        self.live.copy_(self.host, non_blocking=True)
        self.next.copy_(self.host, non_blocking=True)
        engine.h2d_bytes += self.host.numel() * 4

    def choose(self, logits, scores, behind_prompt: bool = False) -> None:
        """From the logits behind every beam to the next step's description.  Behind the prompt every beam goes on from the first, which alone holds it: also those of a search that is
        over or has too few candidates, which are run forward beside the others like any row."""
        p, (step, slots, pages, tables) = self.params, self.now
        made, new_slots, new_pages, new_tables = self.then
        found = ops.beam_candidates(logits, scores, p.keep)
        ops.beam_advance(*found, step.pool, step.lengths, step.done, beams=p.beams, stop_ids=self.stop_ids, max_new=p.max_new,
                         length_penalty=p.length_penalty, out=made)
        ops.beam_reorder(self.first if behind_prompt else made.parents, slots, tables.ctx_len, states=self.states,
                         paged=[(s, t, st) for s, t, st in zip(self.storage, pages, self.strides)], out=(new_slots, new_pages))
        ops.step_tables(self.ones, tables.ctx_len, new_pages, page_size=self.page_size, num_tokens=self.R, strides=self.strides, out=new_tables)
        self.live.copy_(self.next)

    def run(self, engine: Engine) -> None:
        """One step of every search."""
        def train():
            self.choose(engine.model.forward(self.ctx, engine.layer_caches), self.now[0].scores)
        if engine.device.type != "cuda" or not self.graphed:
            train()
        elif self.graph is None:
            before = ops.launches["own"]
            train()
            self.launches = ops.launches["own"] - before
            self.graph, self.reporting = captured(train, self.launches)
        else:
            self.graph.replay()
            ops.launches["own"] += self.launches
            ops.note_status_word_launches(self.reporting)
        engine.steps_run += 1

    graphed = True


class BeamSearch:
    """Searches on an engine, which other requests may share: only the pages and slots that are free are taken, and all come back."""

    KEPT = 4               # shapes (searches, parameters, context) whose buffers and graph are kept

    def __init__(self, engine: Engine, *, chunk_size: int = 512, max_batch_tokens: int = 2048, cuda_graphs: bool = True):
        self.engine = engine
        self.chunk_size, self.max_batch_tokens = int(chunk_size), int(max_batch_tokens)
        self.cuda_graphs = bool(cuda_graphs)
        self._kept: "OrderedDict[tuple, _Searches]" = OrderedDict()
        self._calls = 0

    def search(self, prompts, params: BeamParams | None = None) -> list:
        """Per prompt (a list of token ids), its `BeamResult`s, best first.  Prompts that fit side by side run side by side; where one fits in no case, none runs."""
        params = replace(params or BeamParams())         # (checked again, and ours: the kept graphs are made for it)
        prompts = [[int(t) for t in p] for p in prompts]
        eng = self.engine
        for p in prompts:
            if not p:
                raise ValueError("a request needs at least one prompt token")
            if len(p) + params.max_new > eng.max_positions:
                raise ValueError(f"prompt ({len(p)}) + max_new ({params.max_new}) exceeds the model's {eng.max_positions} positions")
            if min(p) < 0 or max(p) >= eng.vocab_size:
                raise ValueError("a prompt's token id is outside the vocabulary")
        if any(not 0 <= s < eng.vocab_size for s in params.stop_ids):
            raise ValueError("a stop id is outside the vocabulary")
        for p in prompts:                         # each by itself fits what is free, before any of them runs (it all comes back between them)
            self._fitting([p], params)
        results, at = [], 0
        while at < len(prompts):
            n = self._fitting(prompts[at:], params)
            results += self._side_by_side(prompts[at:at + n], params)
            at += n
        return results

    def _fitting(self, prompts, params) -> int:
        """How many of the prompts, from the first on, the free slots and pages hold at once."""
        cache = self.engine.cache
        room = [g.pool.free_count for g in cache.groups]
        n = 0
        for p in prompts[:min(cache.slots.free_count // params.beams, ops.MAX_BEAM_ROWS // params.beams)]:
            need = []
            for gi, g in enumerate(cache.groups):
                total = cache.pages_for(len(p) + params.max_new, gi)
                need.append(total + (params.beams - 1) * (total - len(p) // g.need.stride // cache.page_size))
            if any(a > b for a, b in zip(need, room)):
                break
            room = [b - a for a, b in zip(need, room)]
            n += 1
        if n == 0:
            raise OutOfPages(f"a search of {params.beams} beams over {len(prompts[0])} + {params.max_new} tokens needs more state slots or pages than are free "
                             f"({cache.slots.free_count} slots, {room} pages)")
        return n

    def _side_by_side(self, prompts, params) -> list:
        eng, cache, B = self.engine, self.engine.cache, params.beams
        self._calls += 1
        ids = [("beam search", id(self), self._calls, g) for g in range(len(prompts))]
        taken = []
        try:
            logits = self._prompts(ids, prompts, params, taken)
            rows = []
            for g, p in enumerate(prompts):
                rows.append(cache.requests[ids[g]])
                for b in range(1, B):
                    rows.append(cache.fork_request(ids[g], ids[g] + (b,), len(p) + params.max_new))
                    taken.append(ids[g] + (b,))
            return self._steps(rows, logits, prompts, params)
        finally:
            if eng.device.type == "cuda":
                torch.cuda.current_stream(eng.device).synchronize()        # nothing in flight reads what goes back
            for r in reversed(taken):
                cache.free_request(r)

    def _prompts(self, ids, prompts, params, taken) -> torch.Tensor:
        """The prompts' portions; the logits behind each prompt, ``[G, V]``."""
        eng, cache = self.engine, self.engine.cache
        for r, p in zip(ids, prompts):
            cache.add_request(r)
            taken.append(r)
            cache.reserve(r, len(p) + params.max_new)
        done, logits = [0] * len(prompts), [None] * len(prompts)
        while any(d < len(p) for d, p in zip(done, prompts)):
            budget, entries, last = self.max_batch_tokens, [], []
            for g, p in enumerate(prompts):
                n = min(len(p) - done[g], self.chunk_size, budget)
                if n > 0:
                    ends = done[g] + n == len(p)
                    entries.append(StepEntry(ids[g], p[done[g]:done[g] + n], [n - 1] if ends else []))
                    if ends:
                        last.append(g)
                    done[g] += n
                    budget -= n
            got = eng.step(entries)
            for i, g in enumerate(last):
                logits[g] = got[i:i + 1]
        return torch.cat(logits) if len(logits) > 1 else logits[0].contiguous()

    def _steps(self, rows, logits, prompts, params) -> list:
        eng, G, B, W = self.engine, len(prompts), params.beams, params.results
        s = self._searches(G, params, DecodeGraphs.bucket(max(len(p) for p in prompts) + params.max_new))
        s.begin(eng, rows)
        a, z = s.back
        pin = eng.device.type == "cuda"
        back = torch.zeros((params.max_new, z - a), dtype=torch.int32, pin_memory=pin)
        ready = []

        def note(t):
            back[t].copy_(s.live[a:z], non_blocking=True)
            if pin:
                ready.append(torch.cuda.Event())
                ready[t].record()

        def over(t):
            if pin:
                ready[t].synchronize()
            lo = s.layout.offs["done"] - a
            return bool(back[t, lo:lo + G].all())
        # before the first token there is one beam a search, of score 0
        s.choose(logits, torch.zeros((G, 1), dtype=torch.float32, device=eng.device), behind_prompt=True)
        note(0)
        steps = 1
        while steps < params.max_new:
            if steps > 1 and over(steps - 2):      # (the step just queued is not waited for)
                break
            s.run(eng)
            note(steps)
            steps += 1
        step = s.now[0]
        pool = [x.cpu().numpy() for x in step.pool]
        if pin:
            ops.check_tcgen05_status()
        history = back[:steps].numpy()
        tokens = history[:, :G * B].reshape(steps, G, B)
        lo = s.layout.offs["parents"] - a
        parents = history[:, lo:lo + G * B].reshape(steps, G, B)
        out = []
        for g in range(G):
            found = []
            for score, n, beam, token in zip(*(x[g].tolist() for x in pool)):
                if score == -np.inf:
                    break
                ids, stop = [], token in params.stop_ids
                for t in range(n - 2, -1, -1):     # the beams behind the n-th token, from the last
                    ids.append(int(tokens[t, g, beam]))
                    beam = int(parents[t, g, beam])
                ids.reverse()
                found.append(BeamResult(ids if stop else ids + [token], score, "stop" if stop else "length"))
            out.append(found)
        return out

    def _searches(self, G: int, params: BeamParams, bucket: int) -> _Searches:
        bucket = min(bucket, self.engine.max_positions)
        key = (G, params.beams, params.results, params.max_new, params.length_penalty, params.stop_ids, bucket)
        s = self._kept.pop(key, None)
        if s is None:
            s = _Searches(self.engine, G, params, bucket)
            s.graphed = self.cuda_graphs
            while len(self._kept) >= self.KEPT:
                self._kept.popitem(last=False)
        self._kept[key] = s
        return s
