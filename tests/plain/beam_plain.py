"""Beam search in numpy and float64, one search, beam and token at a time: what the operators have to give, and a whole search over a plain model's logits.
`CPU_OPS` are the operators over CPU tensors, for engine logic without a GPU."""

from __future__ import annotations

import numpy as np
import torch


def log_softmax(row):
    """float64 log-probabilities of one row; what is not a number counts as minus infinity, an infinite maximum takes all mass.  None: the row offers nothing."""
    x = np.asarray(row, dtype=np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return None
    d = np.full_like(x, -np.inf)
    np.subtract(x, top, out=d, where=(x < top) & (top < np.inf))
    d[x == top] = 0.0
    return d - np.log(np.exp(d).sum())


def candidates(logits, scores, keep):
    """[(score float64, beam, token)] of one search, at most ``keep``: by score, then beam, then logit, then token."""
    found = []
    for b, row in enumerate(logits):
        row = np.asarray(row, dtype=np.float64)
        lp = log_softmax(row)
        if lp is None or not scores[b] > -np.inf:
            continue
        order = sorted(range(len(row)), key=lambda t: (-row[t] if not np.isnan(row[t]) else np.inf, t))[:keep]
        found += [(float(scores[b]) + lp[t], b, -row[t], t) for t in order if lp[t] > -np.inf]
    found.sort(key=lambda c: (-c[0],) + c[1:])
    return [(s, b, t) for s, b, _, t in found[:keep]]


def norms(s, n, power):
    """The float32 values that ``s / n ** power`` may have: the rounding of the float64 quotient, and where that lies within 2^-50 (relative) of the midpoint of two float32 values
    both of them.  A float64 power is good to 2 units (2^-51), the division to half a unit more, so another float64 library's quotient differs by less than 2^-50 and rounds to another
    float32 only across such a midpoint (0.1 rounded to float32, times 3, is one exactly: a power of -1/2 at n = 9)."""
    q = np.float64(s) / np.float64(n) ** np.float64(power)
    return sorted({np.float32(q), np.float32(q * (1 - 2.0 ** -50)), np.float32(q * (1 + 2.0 ** -50))})


def advance(cands, pool, length, done, *, beams, stop_ids, max_new, power, width, seen=()):
    """One search's step: (next [(score, parent, token)], pool [(norm, length, parent, token)], length, done), scores rounded to float32.  ``seen``: float32 scores among which the one
    is taken where two are right (`norms`)."""
    idle = [(-np.inf, i, 0) for i in range(beams)]
    pool = list(pool)
    if done:
        return idle, pool, length, 1
    n = length + 1

    def norm(s, at):
        either = norms(s, at, power)
        return next((v for v in either if len(either) > 1 and v in seen), np.float32(np.float64(s) / np.float64(at) ** np.float64(power)))

    def enter(s, parent, token):
        v = norm(s, n)
        at = sum(p[0] >= v for p in pool)
        pool.insert(at, (v, n, parent, token))
        del pool[width:]
    live = []
    for r, (s, b, t) in enumerate(cands):
        if not s > -np.inf:
            continue
        if t in stop_ids:
            if r < beams:
                enter(s, b, t)
        elif len(live) < beams:
            live.append((s, b, t))
    over = not live
    if n >= max_new:
        for c in live:
            enter(*c)
        over = True
    if live and len(pool) == width and norm(live[0][0], max_new if power >= 0 else n + 1) <= pool[-1][0]:
        over = True
    if over:
        return idle, pool, n, 1
    return live + [(-np.inf, -1, 0)] * (beams - len(live)), pool, n, 0


def places(parents):
    """(source row, taken row, copied) of each beam of one search."""
    B = len(parents)
    spare = [b for b in range(B) if b not in parents]
    out, seen = [], set()
    for p in parents:
        if 0 <= p < B and p not in seen:
            seen.add(p)
            out.append((p, p, False))
        else:
            t = spare.pop(0)
            out.append((p if 0 <= p < B else t, t, 0 <= p < B))
    return out


def reorder(parents, slots, lens, states, paged):
    """In place on copies the caller made: (new slots, new tables)."""
    G, B = parents.shape
    new_slots, tables = slots.copy(), [t.copy() for _, t, _ in paged]
    for g in range(G):
        for i, (src, takes, copied) in enumerate(places(list(parents[g]))):
            r, src, takes = g * B + i, g * B + src, g * B + takes
            new_slots[r] = slots[takes]
            if copied:
                for s in states:
                    s[slots[takes]] = s[slots[src]]
            for (storage, table, stride), new in zip(paged, tables):
                ps = storage.shape[-2]
                entries = lens[g] // stride
                at, written = entries // ps, entries % ps
                new[r, :at] = table[src, :at]
                if written and at < table.shape[1]:
                    new[r, at] = table[takes, at]
                    a, b = table[src, at], table[takes, at]
                    if copied and a >= 0 and b >= 0:
                        storage[..., b, :, :written, :] = storage[..., a, :, :written, :]
    return new_slots, tables


def step_tables(q_lens, have, page_tables, *, page_size, num_tokens, strides, rows, free, columns):
    """(q_start, ctx_len, positions, seq_of_token, block tables, slot mappings); ``page_tables`` grow in place."""
    S, T = len(q_lens), num_tokens
    q_start = np.minimum(np.concatenate([[0], np.cumsum(q_lens)]), T)
    positions, seq = np.zeros(T, dtype=np.int64), np.zeros(T, dtype=np.int64)
    for s in range(S):
        n = q_start[s + 1] - q_start[s]
        positions[q_start[s]:q_start[s + 1]] = have[s] + np.arange(n)
        seq[q_start[s]:q_start[s + 1]] = s
    blocks, maps = [], []
    for k, table in enumerate(page_tables):
        stride, used = strides[k], 0
        bt, sm = np.full((S, columns[k]), -1), np.full(T, -1)
        for s in range(S):
            had, needs = -(-(have[s] // stride) // page_size), -(-((have[s] + q_lens[s]) // stride) // page_size)
            row = table[rows[s]]
            if free[k] is not None:
                for c in range(had, needs):
                    if c < table.shape[1]:
                        row[c] = free[k][used] if used < len(free[k]) else -1
                    used += 1
            m = min(needs, columns[k], table.shape[1])
            bt[s, :m] = row[:m]
            for t in range(q_start[s], q_start[s + 1]):
                p = have[s] + t - q_start[s]
                if (p + 1) % stride == 0:
                    e = (p + 1) // stride - 1
                    page = row[e // page_size] if e // page_size < table.shape[1] else -1
                    sm[t] = page * page_size + e % page_size if page >= 0 else -1
        blocks.append(bt)
        maps.append(sm)
    return q_start, have + q_lens, positions, seq, blocks, maps


def search(logits_of, prompt, *, beams, max_new, stop_ids=(), power=1.0, width=None):
    """A whole search: ``logits_of(ids)`` gives the logits after ``ids``.  [(ids, norm, reason)], best first."""
    width = width or beams
    keep = beams * (1 + len(stop_ids))
    live, pool, length, done = [(0.0, [])], [], 0, 0
    history = {}
    while not done:
        logits = [logits_of(list(prompt) + ids) for _, ids in live]
        c = [(np.float32(s), b, t) for s, b, t in candidates(logits, [s for s, _ in live], keep)]
        nxt, pool, length, done = advance(c, pool, length, done, beams=beams, stop_ids=stop_ids, max_new=max_new, power=power, width=width)
        for e in pool:
            if e[1] == length:
                history.setdefault(e[1:], live[e[2]][1] + ([] if e[3] in stop_ids else [e[3]]))
        live = [(s, live[p][1] + [t]) for s, p, t in nxt if s > -np.inf]
    return [(history[e[1:]], float(e[0]), "stop" if e[3] in stop_ids else "length") for e in pool]


# ---- the operators over CPU tensors ---------------------------------------------------------------------------------------

def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32))


def _put(out, values):
    if out is None:
        return values
    out.copy_(values)
    return out


def beam_candidates(logits, scores, keep):
    (G, B) = scores.shape
    s, p, t = np.full((G, keep), -np.inf, np.float32), np.full((G, keep), -1), np.full((G, keep), -1)
    rows = logits.float().numpy().reshape(G, B, -1)
    for g in range(G):
        for i, c in enumerate(candidates(rows[g], scores[g].numpy(), keep)):
            s[g, i], p[g, i], t[g, i] = c
    return torch.from_numpy(s), _i32(p), _i32(t)


def beam_pool(searches, width, device):
    return _ops().BeamPool(torch.full((searches, width), -float("inf")), *(torch.zeros((searches, width), dtype=torch.int32) for _ in range(3)))


def _ops():
    import sllm_b200.ops as ops
    return ops


def beam_advance(scores, parents, tokens, pool, lengths, done, *, beams, stop_ids=None, max_new, length_penalty=1.0, out=None):
    ops = _ops()
    G, W = pool.scores.shape
    stops = set(stop_ids.tolist()) if stop_ids is not None else set()
    nxt, after, n, over = [], [], [], []
    for g in range(G):
        held = [(np.float32(s), *x) for s, *x in zip(*(p[g].tolist() for p in pool)) if s > -np.inf]
        a, b, c, d = advance(list(zip(scores[g].numpy(), parents[g].tolist(), tokens[g].tolist())), held, int(lengths[g]), int(done[g]), beams=beams, stop_ids=stops,
                             max_new=max_new, power=length_penalty, width=W)
        nxt.append(a)
        after.append(b + [(-np.inf, 0, 0, 0)] * (W - len(b)))
        n.append(c)
        over.append(d)

    def column(rows, i, dtype):
        return torch.tensor([[x[i] for x in r] for r in rows], dtype=dtype)
    f, w = torch.float32, torch.int32
    got = (column(nxt, 0, f), column(nxt, 1, w), column(nxt, 2, w), torch.tensor(n, dtype=w), torch.tensor(over, dtype=w))
    kept = (column(after, 0, f), column(after, 1, w), column(after, 2, w), column(after, 3, w))
    o, op = (out[:5], out.pool) if out is not None else ((None,) * 5, (None,) * 4)
    return ops.BeamStep(*(_put(a, b) for a, b in zip(o, got)), ops.BeamPool(*(_put(a, b) for a, b in zip(op, kept))))


def beam_reorder(parents, slots, lens, *, states=(), paged=(), out=None):
    paged = [(s.numpy() if s.dtype != torch.bfloat16 else s.view(torch.int16).numpy(), t.numpy(), st) for s, t, st in paged]
    new_slots, tables = reorder(parents.numpy(), slots.numpy(), lens.numpy()[::max(1, lens.numel() // max(1, parents.shape[0]))], [s.numpy() for s in states], paged)
    o = out if out is not None else (None, [None] * len(tables))
    return _put(o[0], _i32(new_slots)), [_put(a, _i32(b)) for a, b in zip(o[1], tables)]


def step_tables_op(q_lens, have, page_tables, *, page_size, num_tokens, strides=None, rows=None, free=None, columns=None, out=None):
    n = len(page_tables)
    got = step_tables(q_lens.numpy().astype(np.int64), have.numpy().astype(np.int64), [t.numpy() for t in page_tables], page_size=page_size, num_tokens=num_tokens,
                      strides=strides or [1] * n, rows=rows.numpy() if rows is not None else np.arange(len(q_lens)), free=[None if f is None else f.numpy() for f in free] if free else [None] * n,
                      columns=[t.shape[1] if c is None else c for t, c in zip(page_tables, columns or [None] * n)])
    flat = [_i32(x) for x in got[:4]] + [_i32(x) for x in got[4]] + [_i32(x) for x in got[5]]
    if out is not None:
        flat = [_put(a, b) for a, b in zip((*out[:4], *out.block_tables, *out.slot_mappings), flat)]
    return _ops().StepTables(*flat[:4], tuple(flat[4:4 + n]), tuple(flat[4 + n:]))


CPU_OPS = {"beam_candidates": beam_candidates, "beam_pool": beam_pool, "beam_advance": beam_advance, "beam_reorder": beam_reorder, "step_tables": step_tables_op}
