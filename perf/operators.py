"""The operators of a beam search on the device, beside their plain forms.

A search keeps ``beams`` continuations of a prompt alive.  One step of it, behind the model's logits, is four operators:

* ``candidates``: the best ``keep`` continuations over all beams and the whole vocabulary, by cumulative log-probability;
* ``advance``: which of them go on, which are finished, and whether the search is over;
* ``reorder``: states and pages follow the beams that go on: a parent's first child keeps what the parent has, the others get
  copies of it in the places of beams that have no child;
* ``tables``: the next step's description (starts, positions, slot maps, block tables) from the requests' lengths.

Sizes are those of Qwen2.5-0.5B and 7B (vocabulary, layers, key/value heads) and of the wide recurrent layers of the
side-by-side workloads, in pages of 16 tokens.  The plain forms below are torch's elementary operations.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

PAGE = 16
DEVICE = "cuda"


# ---- the cases ----------------------------------------------------------------------------------------------------------

def _candidates(name, searches, beams, vocab, dtype="float32", stops=1, masked=0.0):
    """``stops``: stop ids, each of which may take a candidate a beam; ``masked``: the share of logits that a grammar rules out."""
    return {"name": name, "op": "candidates", "searches": searches, "beams": beams, "vocab": vocab, "keep": beams * (1 + stops),
            "dtype": dtype, "masked": masked}


def _advance(name, searches, beams, stops, power, late):
    """``late``: the pools hold finished continuations already."""
    return {"name": name, "op": "advance", "searches": searches, "beams": beams, "stops": stops, "keep": beams * (1 + stops),
            "power": power, "late": late}


def _reorder(name, searches, beams, extra, context, runs, heads, dim, layers=0, state_heads=0, state_dim=0, dtype="bfloat16"):
    """``extra``: beams of each search that are a second or later child.  ``runs`` x ``heads`` x ``dim``: keys and values in pages;
    ``layers`` x ``state_heads`` x ``state_dim``^2: float32 states."""
    return {"name": name, "op": "reorder", "searches": searches, "beams": beams, "extra": extra, "context": context, "runs": runs,
            "heads": heads, "dim": dim, "layers": layers, "state_heads": state_heads, "state_dim": state_dim, "dtype": dtype}


def _tables(name, requests, tokens, context, columns, stride=0, grow=False):
    """``tokens``: new tokens of all requests together; ``context``: the longest number of tokens a request has before; ``stride``:
    a second group of pages with an entry per so many tokens; ``grow``: new pages come from a list of free ones."""
    return {"name": name, "op": "tables", "requests": requests, "tokens": tokens, "context": context, "columns": columns,
            "stride": stride, "grow": grow}


def listed():
    return [
        # a tiny model's search: nothing but latency
        _candidates("candidates tiny", 1, 4, 260),
        # one prompt on the small model, logits as the head writes them
        _candidates("candidates 0.5b one prompt", 1, 4, 151936),
        # a few prompts, an odd vocabulary, two stop ids, a grammar that rules out most tokens
        _candidates("candidates ragged masked", 7, 5, 32001, stops=2, masked=0.6),
        # a full batch of wide searches, logits kept in 16 bits
        _candidates("candidates 7b batch", 64, 8, 152064, dtype="bfloat16"),
        # one search between two decode steps
        _advance("advance one search", 1, 4, 1, 1.0, False),
        # many wide searches near their end, several stop ids
        _advance("advance many", 64, 24, 3, 0.7, True),
        # two beams of the small model: the page that is being written, in 24 layers
        _reorder("reorder 0.5b pages", 1, 2, 1, 139, 24, 2, 64),
        # searches of four beams on the main model
        _reorder("reorder 7b pages", 16, 4, 2, 509, 28, 4, 128),
        # the same over recurrent layers with a matrix a head: large states, no pages to speak of
        _reorder("reorder states", 8, 4, 2, 200, 1, 1, 128, layers=8, state_heads=32, state_dim=128),
        # a decode step of a few requests
        _tables("tables decode", 8, 8, 4096, 512),
        # prompt portions of many requests beside decoded tokens, pages taken as they are needed, a second group of pooled entries
        _tables("tables portions", 48, 4099, 2000, 256, stride=4, grow=True),
        # the largest serving step: hundreds of long requests
        _tables("tables long", 512, 32768, 32000, 2100),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"]


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("candidates", "candidates", "advance", "reorder", "reorder", "tables"))
        if op == "candidates":
            case = _candidates("", _log(rng, 1, 64), _log(rng, 1, 24), _log(rng, 64, 152064), rng.choice(("float32", "bfloat16")),
                               rng.randint(0, 2), rng.choice((0.0, 0.0, 0.5, 0.95)))
        elif op == "advance":
            stops = rng.randint(0, 3)
            case = _advance("", _log(rng, 1, 96), _log(rng, 1, 32), stops, round(rng.uniform(-0.5, 2.0), 3), rng.random() < 0.5)
        elif op == "reorder":
            beams = _log(rng, 1, 12)
            state = rng.random() < 0.5
            case = _reorder("", _log(rng, 1, 24), beams, rng.randint(0, beams - 1), _log(rng, 1, 3000), rng.randint(1, 28), rng.choice((1, 2, 4, 7)),
                            rng.choice((20, 64, 128)), *((rng.randint(1, 8), _log(rng, 1, 32), rng.choice((33, 64, 128))) if state else (0, 0, 0)),
                            dtype=rng.choice(("bfloat16", "float32")))
            if _held(case) > 1.2e9:
                continue
        else:
            requests = _log(rng, 1, 512)
            context = _log(rng, 1, 32000)
            tokens = requests if rng.random() < 0.4 else requests + _log(rng, 1, 16384)
            case = _tables("", requests, tokens, context, -(-(context + tokens) // PAGE) + rng.randint(0, 40), rng.choice((0, 0, 4, 7)), rng.random() < 0.5)
            if requests * case["columns"] > 512 * 4100:
                continue
        if case.get("keep", 1) > 128 or _cost(case) > most:
            continue
        del case["name"]
        return case


def _held(case):
    """Bytes that a reorder's caches hold."""
    size = 2 if case["dtype"] == "bfloat16" else 4
    pages = 2 * case["runs"] * _num_pages(case) * case["heads"] * PAGE * case["dim"] * size
    return pages + case["layers"] * (case["searches"] * case["beams"] + 1) * case["state_heads"] * case["state_dim"] ** 2 * 4


def _num_pages(case):
    """The prompt's whole pages once a search, three further ones a beam, and some that nobody holds."""
    return case["searches"] * (case["context"] // PAGE + 3 * case["beams"]) + 5


def work(case):
    """Bytes: every input once, every output once."""
    op = case["op"]
    if op == "candidates":
        n = case["searches"] * case["beams"] * case["vocab"]
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": n * size + 4 * case["searches"] * (case["beams"] + 3 * case["keep"]), "flops": 4 * n}
    if op == "advance":
        g, b = case["searches"], case["beams"]
        return {"bytes": 4 * g * (3 * case["keep"] + 2 * 4 * b + 3 * b + 4) + 4 * case["stops"], "flops": 0}
    if op == "reorder":
        rows = case["searches"] * case["beams"]
        copies = case["searches"] * case["extra"]
        size = 2 if case["dtype"] == "bfloat16" else 4
        page = 2 * case["runs"] * case["heads"] * (case["context"] % PAGE) * case["dim"] * size
        state = case["layers"] * case["state_heads"] * case["state_dim"] ** 2 * 4
        return {"bytes": 2 * copies * (page + state) + 4 * rows * (2 * (case["context"] // PAGE + 3) + 3), "flops": 0}
    groups = 2 if case["stride"] else 1
    s, t = case["requests"], case["tokens"]
    used = s * (case["context"] // 2 // PAGE + 1)          # (requests have from one token to `context`)
    return {"bytes": 4 * (2 * s + (2 * s + 1) + 2 * t + groups * (t + s * case["columns"]) + used), "flops": 0}


# ---- inputs ---------------------------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _int32(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device=DEVICE)


def _candidates_inputs(case, seed):
    g = _generator(seed)
    G, B, V = case["searches"], case["beams"], case["vocab"]
    # the beams of a search are alike: a part of the logits is theirs together
    logits = torch.randn((G, 1, V), generator=g, device=DEVICE) * 1.5 + torch.randn((G, B, V), generator=g, device=DEVICE) * 1.5
    if case["masked"]:
        logits.masked_fill_(torch.rand((G, 1, V), generator=g, device=DEVICE) < case["masked"], -math.inf)
    scores = -torch.rand((G, B), generator=g, device=DEVICE) * 6 - 20
    scores = scores.sort(dim=1, descending=True).values.contiguous()
    if B > 2 and G > 1:
        scores[0, B - 1] = -math.inf                       # a search with a beam less
        logits[1, B - 1] = -math.inf                       # a beam whose every token is ruled out
    return logits.reshape(G * B, V).to(getattr(torch, case["dtype"])), scores


def _advance_inputs(case, seed):
    rng = np.random.default_rng(seed)
    G, B, K = case["searches"], case["beams"], case["keep"]
    stop = 2 + np.arange(case["stops"])
    scores = -np.sort(rng.uniform(5, 30, (G, K)).astype(np.float32), axis=1)
    parents = rng.integers(0, B, (G, K))
    tokens = rng.integers(100, 30000, (G, K))
    if case["stops"]:
        at = rng.random((G, K)) < 0.25
        tokens[at] = rng.choice(stop, int(at.sum()))
    if G > 1:                                              # a search that finds fewer continuations
        scores[1, B:], parents[1, B:], tokens[1, B:] = -np.inf, -1, -1
    lengths = rng.integers(8, 60, G)
    pool_scores = np.full((G, B), -np.inf, np.float32)
    held = np.zeros((G, B), dtype=bool)
    if case["late"]:
        held = np.arange(B)[None] < rng.integers(0, B + 1, (G, 1))
    pool_scores[held] = 0
    finished = -np.sort(rng.uniform(0.2, 1.4, (G, B)).astype(np.float32), axis=1)
    pool_scores = np.where(held, finished, pool_scores).astype(np.float32)
    pool = [np.where(held, v, 0) for v in (rng.integers(1, 8, (G, B)), rng.integers(0, B, (G, B)), rng.integers(2, 30000, (G, B)))]
    done = (rng.random(G) < 0.1) if G > 2 else np.zeros(G, dtype=bool)
    return {"scores": torch.from_numpy(scores).to(DEVICE), "parents": _int32(parents), "tokens": _int32(tokens),
            "pool_scores": torch.from_numpy(pool_scores).to(DEVICE), "pool": [_int32(p) for p in pool], "lengths": _int32(lengths),
            "done": _int32(done), "stop": _int32(stop), "max_new": 56}


def _reorder_inputs(case, seed):
    rng = np.random.default_rng(seed)
    G, B, n = case["searches"], case["beams"], case["context"]
    rows, shared = G * B, case["context"] // PAGE
    dtype = getattr(torch, case["dtype"])
    parents = np.zeros((G, B), dtype=np.int64)
    for i in range(G):
        alive = rng.permutation(B)[:B - case["extra"]]
        parents[i] = rng.permutation(np.concatenate([alive, rng.choice(alive, case["extra"])]))
    pages = rng.permutation(_num_pages(case))
    own_pages = pages[:rows * 3].reshape(rows, 3)
    prompt = pages[rows * 3:rows * 3 + G * shared].reshape(G, shared).repeat(B, axis=0)
    table = np.concatenate([prompt, own_pages], axis=1)
    g = _generator(seed)
    kv = torch.randn((case["runs"], 2, _num_pages(case), case["heads"], PAGE, case["dim"]), generator=g, device=DEVICE, dtype=dtype)
    H, D = case["state_heads"], case["state_dim"]
    states = [torch.randn((rows + 1, H, D, D), generator=g, device=DEVICE) for _ in range(case["layers"])]
    return {"parents": _int32(parents), "slots": _int32(rng.permutation(rows)), "lens": _int32(np.full(G, n)), "table": _int32(table),
            "kv": kv, "states": states}


def _tables_inputs(case, seed):
    rng = np.random.default_rng(seed)
    S, T, MP = case["requests"], case["tokens"], case["columns"]
    q = np.ones(S, dtype=np.int64)
    if T > S:                                              # a few prompt portions take what is not a decoded token
        some = rng.choice(S, max(1, S // 4), replace=False)
        q[some] += rng.multinomial(T - S, np.full(some.size, 1 / some.size))
    have = np.maximum(1, np.exp(rng.uniform(0, math.log(case["context"] + 1), S)).astype(np.int64))
    have[rng.integers(0, S)] = case["context"]
    most = MP * PAGE - q
    have = np.minimum(have, most)
    have[rng.random(S) < 0.1] = 0                          # requests whose first portion this is
    strides = [1] + ([case["stride"]] if case["stride"] else [])
    tables, free = [], []
    for stride in strides:
        before, after = have // stride, (have + q) // stride
        had, needs = -(-before // PAGE), -(-after // PAGE)
        held = had if case["grow"] else needs
        ids = rng.permutation(int(needs.sum()) + 7)
        table = np.full((S + 3, MP), -1, dtype=np.int64)
        cell = np.arange(MP)[None] < held[:, None]
        table[:S][cell] = ids[:int(held.sum())]
        tables.append(table)
        free.append(ids[int(held.sum()):])
    rows = rng.permutation(S + 3)[:S]                      # requests come and go: a step's are any rows of the table
    for k, table in enumerate(tables):
        placed = np.full_like(table, -1)
        placed[rows] = table[:S]
        tables[k] = placed
    return {"q": _int32(q), "have": _int32(have), "rows": _int32(rows), "tables": [_int32(t) for t in tables],
            "free": [_int32(f) for f in free] if case["grow"] else None, "strides": strides, "tokens": T}


def prepare(case, seed):
    op = case["op"]
    if op == "candidates":
        logits, scores = _candidates_inputs(case, seed)
        state = {"logits": logits, "scores": scores}
    else:
        state = {"advance": _advance_inputs, "reorder": _reorder_inputs, "tables": _tables_inputs}[op](case, seed)
    state["case"] = case
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------------

def run(state):
    return {"candidates": _run_candidates, "advance": _run_advance, "reorder": _run_reorder, "tables": _run_tables}[state["case"]["op"]](state)


def _run_candidates(state):
    logits, scores, keep = state["logits"], state["scores"], state["case"]["keep"]
    if own:
        from sllm_b200 import ops
        s, p, t = ops.beam_candidates(logits, scores, keep)
        return {"scores": s, "parents": p, "tokens": t}
    G, B = scores.shape
    V = logits.shape[1]
    x = logits.reshape(G, B, V).double()                   # in 64 bits: continuations of different beams lie close together
    top = x.amax(dim=2, keepdim=True)
    d = torch.where(x == top, 0.0, x - top)
    d = torch.where(torch.isneginf(top), -math.inf, d)
    lse = d.exp().sum(dim=2, keepdim=True).log()
    # within a beam by logit, then by token; between beams by score, then by beam
    n = min(keep, V)
    order = torch.sort(x, dim=2, descending=True, stable=True).indices[:, :, :n]
    s = torch.gather(d, 2, order) - lse + scores.double()[:, :, None]
    s = torch.where(s > -math.inf, s, -math.inf).reshape(G, B * n)
    best = torch.sort(s, dim=1, descending=True, stable=True)
    m = min(keep, B * n)
    value, at = best.values[:, :m], best.indices[:, :m]
    there = value > -math.inf
    parents = torch.where(there, at // n, -1)
    tokens = torch.where(there, torch.gather(order.reshape(G, B * n), 1, at), -1)
    out = torch.full((G, keep), -math.inf, device=logits.device)
    out_p, out_t = (torch.full((G, keep), -1, dtype=torch.int32, device=logits.device) for _ in range(2))
    out[:, :m], out_p[:, :m], out_t[:, :m] = value.float(), parents.int(), tokens.int()
    return {"scores": out, "parents": out_p, "tokens": out_t}


def _run_advance(state):
    case = state["case"]
    W, B, K = case["beams"], case["beams"], case["keep"]
    if own:
        from sllm_b200 import ops
        pool = ops.BeamPool(state["pool_scores"], *state["pool"])
        step = ops.beam_advance(state["scores"], state["parents"], state["tokens"], pool, state["lengths"], state["done"], beams=B,
                                stop_ids=state["stop"], max_new=state["max_new"], length_penalty=case["power"])
        return {"scores": step.scores, "parents": step.parents, "tokens": step.tokens, "lengths": step.lengths, "done": step.done,
                "pool": list(step.pool)}
    s, parents, tokens = state["scores"], state["parents"].long(), state["tokens"].long()
    G, power, max_new = s.shape[0], case["power"], state["max_new"]
    dev = s.device
    was_done = state["done"].bool()
    length = state["lengths"].long() + 1
    at_end = length >= max_new
    there = s > -math.inf
    stops = (tokens[:, :, None] == state["stop"].long()[None, None, :]).any(dim=2) & there
    live = there & ~stops
    order = torch.cumsum(live, dim=1)
    live = live & (order <= B)
    # what enters the pool: stops among the first B candidates, and at the last length what lives, behind them
    norm = (s.double() / length.double()[:, None] ** power).float()
    rank = torch.arange(K, device=dev)[None].expand(G, K)
    enters = torch.cat([stops & (rank < B), live & at_end[:, None]], dim=1)
    new = [torch.cat([v, v], dim=1) for v in (norm, length[:, None].expand(G, K), parents, tokens)]
    new_score = torch.where(enters & ~was_done[:, None], new[0], -math.inf)
    all_scores = torch.cat([state["pool_scores"], new_score], dim=1)
    best = torch.sort(all_scores, dim=1, descending=True, stable=True).indices[:, :W]
    pool = [torch.gather(all_scores, 1, best)]
    empty = pool[0] == -math.inf
    for held, v in zip(state["pool"], new[1:]):
        pool.append(torch.where(empty, 0, torch.gather(torch.cat([held.long(), v], dim=1), 1, best)).int())
    # over: at the last length, with nothing alive, or when the best that lives cannot displace the worst of a full pool
    lead = torch.where(live, s, -math.inf).amax(dim=1).double()
    reach = torch.full_like(length, max_new) if power >= 0 else length + 1
    bound = (lead / reach.double() ** power).float()
    over = was_done | at_end | ~live.any(dim=1) | ((pool[0][:, W - 1] > -math.inf) & (bound <= pool[0][:, W - 1]))
    # the beams that go on, in the candidates' order
    first = torch.sort((~live).int(), dim=1, stable=True).indices[:, :B]
    goes = torch.gather(live, 1, first) & ~over[:, None]
    idle = torch.where(over[:, None], torch.arange(B, device=dev)[None], -1)
    out_s = torch.where(goes, torch.gather(s, 1, first), -math.inf)
    out_p = torch.where(goes, torch.gather(parents, 1, first), idle).int()
    out_t = torch.where(goes, torch.gather(tokens, 1, first), 0).int()
    lengths = torch.where(was_done, state["lengths"].long(), length).int()
    return {"scores": out_s, "parents": out_p, "tokens": out_t, "lengths": lengths, "done": over.int(), "pool": pool}


def _run_reorder(state):
    if own:
        from sllm_b200 import ops
        slots, tables = ops.beam_reorder(state["parents"], state["slots"], state["lens"], states=state["states"],
                                         paged=[(state["kv"], state["table"], 1)])
        return {"slots": slots, "tables": tables, "states": state["states"], "kv": state["kv"]}
    parents = state["parents"].long()
    G, B = parents.shape
    dev = parents.device
    same = parents[:, :, None] == parents[:, None, :]
    earlier = torch.ones((B, B), dtype=torch.bool, device=dev).tril(-1)
    keeps = ~(same & earlier).any(dim=2) & (parents >= 0)
    childless = ~(parents[:, None, :] == torch.arange(B, device=dev)[None, :, None]).any(dim=2)
    spare = torch.sort((~childless).int(), dim=1, stable=True).indices          # beams without a child, in order, first
    nth = torch.cumsum(~keeps, dim=1) - 1
    takes = torch.where(keeps, parents, torch.gather(spare, 1, nth.clamp(min=0)))
    base = torch.arange(G, device=dev)[:, None] * B
    source = (torch.where(parents >= 0, parents, takes) + base).reshape(-1)
    takes = (takes + base).reshape(-1)
    slots = state["slots"].long()
    for t in state["states"]:
        t[slots[takes]] = t[slots[source]]
    table = state["table"]
    lens = state["lens"].long()[:, None].expand(G, B).reshape(-1)
    at = (lens // PAGE)[:, None]
    col = torch.arange(table.shape[1], device=dev)[None]
    begun = (lens % PAGE > 0)[:, None]
    new = torch.where(col < at, table[source], torch.where((col == at) & begun, table[takes], table))
    src = torch.gather(table[source], 1, at).reshape(-1).long()
    dst = torch.gather(new, 1, at).reshape(-1).long()
    kv, fill = state["kv"], (lens % PAGE)[:, None]
    written = (torch.arange(PAGE, device=dev)[None] < fill)[None, None, :, None, :, None]
    kv[:, :, dst] = torch.where(written, kv[:, :, src], kv[:, :, dst])
    return {"slots": slots[takes].int(), "tables": [new], "states": state["states"], "kv": kv}


def _run_tables(state):
    case, T = state["case"], state["tokens"]
    if own:
        from sllm_b200 import ops
        t = ops.step_tables(state["q"], state["have"], state["tables"], page_size=PAGE, num_tokens=T, strides=state["strides"],
                            rows=state["rows"], free=state["free"])
        return {"q_start": t.q_start, "ctx_len": t.ctx_len, "positions": t.positions, "seq_of_token": t.seq_of_token,
                "block_tables": list(t.block_tables), "slot_mappings": list(t.slot_mappings),
                "page_tables": state["tables"] if state["free"] is not None else []}
    q, have, rows = state["q"].long(), state["have"].long(), state["rows"].long()
    S = q.shape[0]
    dev = q.device
    ends = torch.cumsum(q, 0)
    q_start = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), ends])
    ctx = have + q
    token = torch.arange(T, device=dev)
    seq = torch.searchsorted(ends, token, right=True)
    position = token - q_start[seq] + have[seq]
    tables, maps = [], []
    for k, stride in enumerate(state["strides"]):
        page_table = state["tables"][k]
        MP = page_table.shape[1]
        col = torch.arange(MP, device=dev)[None]
        had, needs = -(-(have // stride) // PAGE), -(-(ctx // stride) // PAGE)
        table = page_table[rows].long()
        if state["free"] is not None:
            free = state["free"][k].long()
            fresh = torch.cumsum(needs - had, 0) - (needs - had)
            which = (fresh[:, None] + col - had[:, None]).clamp(0, free.shape[0] - 1)
            table = torch.where((col >= had[:, None]) & (col < needs[:, None]), free[which], table)
            page_table[rows] = table.int()
        tables.append(torch.where(col < needs[:, None], table, -1).int())
        entry = position if stride == 1 else (position + 1) // stride - 1
        writes = torch.ones_like(entry, dtype=torch.bool) if stride == 1 else (position + 1) % stride == 0
        entry = entry.clamp(min=0)
        page = table[seq, (entry // PAGE).clamp(max=MP - 1)]
        maps.append(torch.where(writes & (page >= 0), page * PAGE + entry % PAGE, -1).int())
    return {"q_start": q_start.int(), "ctx_len": ctx.int(), "positions": position.int(), "seq_of_token": seq.int(),
            "block_tables": tables, "slot_mappings": maps, "page_tables": state["tables"] if state["free"] is not None else []}


# ---- the same in 64 bits, from the definition -----------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "candidates":
        return _exact_candidates(case, seed)
    if case["op"] == "advance":
        return _exact_advance(case, seed)
    return None                                            # copies and whole numbers


def _exact_candidates(case, seed):
    logits, scores = _candidates_inputs(case, seed)
    logits, scores = logits.float().cpu().numpy(), scores.cpu().numpy().astype(np.float64)
    G, B = scores.shape
    V, keep = logits.shape[1], case["keep"]
    out = np.full((G, keep), -np.inf)
    for g in range(G):
        found = []
        for b in range(B):
            x = logits[g * B + b].astype(np.float64)
            if not np.isfinite(scores[g, b]) or not (x > -np.inf).any():
                continue
            log_p = x - x.max()
            log_p -= np.log(np.sum(np.exp(log_p)))
            log_p = log_p[log_p > -np.inf]
            found.append(scores[g, b] + (np.partition(log_p, -keep)[-keep:] if log_p.size > keep else log_p))
        best = np.sort(np.concatenate(found))[::-1][:keep] if found else np.zeros(0)
        out[g, :best.size] = best
    return {"scores": out, "parents": None, "tokens": None}


def _exact_advance(case, seed):
    inputs = _advance_inputs(case, seed)
    host = {k: v.cpu().numpy() for k, v in inputs.items() if isinstance(v, torch.Tensor)}
    G, B, K, power, max_new = case["searches"], case["beams"], case["keep"], case["power"], inputs["max_new"]
    stop = set(host["stop"].tolist())
    scores, pools = np.full((G, B), -np.inf), np.full((G, B), -np.inf)
    for g in range(G):
        pool = [float(v) for v in host["pool_scores"][g] if v > -np.inf]
        if host["done"][g]:
            pools[g, :len(pool)] = pool
            continue
        n = int(host["lengths"][g]) + 1
        live = []
        for r in range(K):
            s = float(host["scores"][g, r])
            if s == -math.inf:
                continue
            if int(host["tokens"][g, r]) in stop:
                if r < B:
                    pool.append(s / n ** power)
            elif len(live) < B:
                live.append(s)
        if n >= max_new:
            pool += [s / n ** power for s in live]
        pool = sorted(pool, reverse=True)[:B]
        pools[g, :len(pool)] = pool
        reach = max_new if power >= 0 else n + 1
        if n >= max_new or not live or (len(pool) == B and np.float32(live[0] / reach ** power) <= np.float32(pool[-1])):
            continue
        scores[g, :len(live)] = live
    return {"scores": scores, "parents": None, "tokens": None, "lengths": None, "done": None, "pool": [pools, None, None, None]}


if __name__ == "__main__":
    for c in listed() + [dict(draw(random.Random(i)), name=f"drawn {i}") for i in range(6)]:
        print(c["name"], c, work(c))
