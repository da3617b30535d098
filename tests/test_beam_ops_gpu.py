"""The operators of a beam search against their definitions in float64 (tests/plain/beam_plain.py).  Whole numbers are equal; scores are float32 roundings of a float64 sum whose
only float32 part are the exponentials, see `SCORE`."""

import itertools
import math

import numpy as np
import pytest
import torch

from tests.conftest import cuda_or_skip
from tests.plain import beam_plain as plain

pytestmark = pytest.mark.gpu

# A score s + (d - log sum) is off by the rounding of the result, 2^-24 of it, and by the relative error of the sum of exponentials, in units of 2^-24, which are means under the softmax
# itself, where |x - max| is ln V <= 12 at the most: a thread's exponentials 19 (one rounding of the exponent 12, log2 e's own 3, the hardware's 2^-22 4), its sum 27 (8 additions
# of a batch and up to 19 batches of these rows' parts), the threads' sums brought to one maximum 28 (a difference and a product 12 each, 4): 74.  What follows is 64 bits.
SCORE = lambda s: 2.0 ** -24 * np.abs(s) + 2.0 ** -24 * (19 + 27 + 28)      # noqa: E731


def _i32(a, dev):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=dev)


def _check_candidates(logits, scores, keep, gap=2e-6):
    """Every place of every search.  Where two candidates of different beams lie closer than the scores' own error the order is not tested (the inputs keep away from that but for
    equal rows, which are equal in every bit)."""
    import sllm_b200.ops as ops
    s, p, t = (x.cpu().numpy() for x in ops.beam_candidates(logits, scores, keep))
    G, B = scores.shape
    rows = logits.float().cpu().numpy().reshape(G, B, -1)
    for g in range(G):
        want = plain.candidates(rows[g], scores[g].cpu().numpy(), keep)
        n = len(want)
        assert (s[g, n:] == -np.inf).all() and (p[g, n:] == -1).all() and (t[g, n:] == -1).all()
        if not n:
            continue
        ws, wb, wt = (np.array(x) for x in zip(*want))
        assert (np.abs(s[g, :n] - ws) <= SCORE(ws)).all() or np.array_equal(s[g, :n], ws.astype(np.float32)), (g, np.abs(s[g, :n] - ws).max())
        assert np.array_equal(p[g, :n], wb) and np.array_equal(t[g, :n], wt), (g, np.flatnonzero((p[g, :n] != wb) | (t[g, :n] != wt))[:5])


@pytest.mark.parametrize("V", [1, 3, 260, 1021, 4096, 32001, 151936])
@pytest.mark.parametrize("G,B,keep", [(1, 1, 1), (1, 4, 8), (3, 5, 15), (2, 32, 128), (9, 2, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_candidates(V, G, B, keep, dtype):
    dev = cuda_or_skip()
    g = torch.Generator(device=dev).manual_seed(V + 7 * G + B)
    logits = (torch.randn(G * B, V, device=dev, generator=g) * 3).to(dtype)
    scores = -torch.rand(G, B, device=dev, generator=g) * 5
    _check_candidates(logits, scores, keep)


@pytest.mark.parametrize("V", [40, 5003, 33000])
@pytest.mark.parametrize("keep", [1, 6, 40, 128])
def test_candidates_of_odd_rows(V, keep):
    """Dead beams, masked tokens, rows with nothing, not a number, infinities, ties, sorted rows, equal rows, both zeros."""
    dev = cuda_or_skip()
    g = torch.Generator(device=dev).manual_seed(V + keep)
    G, B = 5, 6
    x = torch.randn(G, B, V, device=dev, generator=g) * 2
    scores = -torch.rand(G, B, device=dev, generator=g) * 5
    scores[0, 1], scores[0, 2] = -math.inf, math.nan
    x[0, 3] = -math.inf
    x[0, 4, ::3] = math.nan
    x[0, 5, : V - 2] = -math.inf
    x[1] = x[1].round()                                        # ties within a row
    x[2, 0] = x[2, 0].sort().values                            # every logit above the ones before
    x[2, 1] = x[2, 1].sort(descending=True).values
    x[2, 2] = 0.0                                              # all equal
    x[2, 3] = torch.finfo(torch.float32).min                   # the type's lowest value everywhere: equal too
    x[2, 4, 1:] = torch.finfo(torch.float32).min               # and behind one that counts
    x[2, 5, 7:9], x[2, 5, 9:11] = -0.0, 0.0
    x[3] = x[3, 0]                                             # equal rows and equal scores: the lower beam first
    scores[3] = scores[3, 0]
    x[4, 0, 5], x[4, 0, V - 1] = math.inf, math.inf            # an infinite maximum takes all
    x[4, 1] = -math.inf
    scores[4, 2:] = -math.inf
    _check_candidates(x.reshape(G * B, V).contiguous(), scores, keep)


def test_candidates_of_rows_off_their_alignment():
    """Rows that begin on any element, a storage that does too."""
    dev = cuda_or_skip()
    for dtype in (torch.float32, torch.bfloat16):
        for V in (5, 1003, 8191):
            for off in (1, 2, 3):
                flat = torch.randn(6 * V + off, device=dev, generator=torch.Generator(device=dev).manual_seed(V + off)).to(dtype)
                _check_candidates(flat[off:].view(6, V), -torch.rand(2, 3, device=dev), 7)


def test_candidates_far_apart_scores_and_large_logits():
    dev = cuda_or_skip()
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn(8, 3001, device=dev, generator=g) * 40 + 500
    scores = torch.tensor([[-3.0, -900.0, -3.5, -40.0], [0.0, -1e-3, -2.0, -5000.0]], device=dev)
    _check_candidates(x, scores, 24)


@pytest.mark.parametrize("V", [7, 1000, 20011])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_candidates_of_rows_of_huge_logits(V, dtype):
    """Rows whose logits are all of a size where float32 has no fractions left (1e4 to the type's end, both signs; a mask of -1e30 everywhere): level ones, ones with a maximum of few, and with a beam of
    ordinary logits beside them."""
    dev = cuda_or_skip()
    sizes = [s * m for m in (1e4, 5e5, 9e5, 2e6, 7e6, 1e8, 1e9, 1e10, 1e20, 1e30, 3e37, 1e38, 3e38) for s in (1, -1)]
    g = torch.Generator(device=dev).manual_seed(V)
    x = torch.empty(len(sizes), 3, V, device=dev)
    for i, m in enumerate(sizes):
        x[i, 0] = m
        x[i, 1] = m * (1 + torch.rand(V, device=dev, generator=g) * 0.1)
        x[i, 1, :: 3] = m if m > 0 else m * 1.1
        x[i, 2] = torch.randn(V, device=dev, generator=g)
    _check_candidates(x.clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).to(dtype).reshape(-1, V).contiguous(), -torch.rand(len(sizes), 3, device=dev, generator=g), 6)


@pytest.mark.parametrize("V", [900, 20011, 70001])
@pytest.mark.parametrize("at", [2907270.0, -2907270.0, 0.0])
def test_candidates_of_rows_across_a_border_of_the_sum(V, at):
    """Logits around +-2^22 / log2 e, where a sum's reference is no whole number any longer, threads and parts of a row on either side of it; and rows with few logits of +-1e7 and 1e30 among
    ordinary ones, early, late and everywhere."""
    dev = cuda_or_skip()
    g = torch.Generator(device=dev).manual_seed(V)
    x = torch.randn(3, 4, V, device=dev, generator=g) * 2 + at
    x[0, 0, : V // 2] -= 7
    x[0, 1, V // 2 :] -= 7
    x[0, 2] = x[0, 2].sort().values
    if at == 0:
        x[1, 0, 3], x[1, 1, V - 1], x[1, 2, V // 2], x[1, 3, ::7] = 1e7, 1e7, 1e30, 1e30
        x[2, 0, : V - 3], x[2, 1, 3:], x[2, 2, ::2], x[2, 3, 1::2] = -1e7, -1e7, -1e30, -3e6
    _check_candidates(x.reshape(12, V), -torch.rand(3, 4, device=dev, generator=g), 5)


@pytest.mark.parametrize("V", [40, 3001, 50000])
@pytest.mark.parametrize("keep", [1, 2, 3, 9])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_beams_whose_best_lie_next_to_each_other(V, keep, dtype):
    """Scores drawn so that the beams' best continuations are equal to some 1e-9, closer than float32 exponentials tell: the order is that of the sums in 64 bits, at the cut too."""
    dev = cuda_or_skip()
    G, B = 40, 3
    g = torch.Generator(device=dev).manual_seed(V + keep)
    logits = (torch.randn(G * B, V, device=dev, generator=g) * 2).to(dtype)
    x = logits.double().reshape(G, B, V)
    best = x.amax(2) - torch.logsumexp(x, 2)
    scores = (best[:, :1] - best).float()
    gaps = (scores.double() + best - best[:, :1]).abs()
    assert gaps.max() < 2e-7                                  # (half a step of scores below 4)
    if keep == 9:
        scores[::2, 2] = -math.inf                            # two of them
    _check_candidates(logits, scores.contiguous(), keep)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", [8.0, 8.5, 9.0, 9.7, 10.3, 11.0, 11.6, 12.2, 13.0, "width 4", "width 6", "width 8", "rising"])
@pytest.mark.parametrize("V", [152064, 152063])
def test_beams_closer_than_sums_in_32_bits_tell_apart(V, kind, dtype):
    """Whole rows (more than the SMs hold blocks) of two beams a search, whose best continuations lie 2^-24 to 2^-16 apart, either first: the order is the one of sums in 64 bits.  One logit above
    equal ones (a number: by how much), where every rounding is the same one; rows of normal logits; rows that rise, whose maximum moves with every batch.  The other beam's row is one
    logit, whose sum is exact, or normal too."""
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    G, B, keep = 160, 2, 2
    g = torch.Generator(device=dev).manual_seed(V)
    x = torch.full((G, B, V), -math.inf, device=dev)
    if isinstance(kind, float):
        x[:, 0] = 3.7 - kind
        x[:, 0, 77] = 3.7
    elif kind == "rising":
        x[:, 0] = torch.arange(V, device=dev) * 1e-5
        x[:, 0, V - 1] += 1.0
    else:
        x[:, 0] = torch.randn(G, V, device=dev, generator=g) * float(kind.split()[1])
    x[:, 1, 5] = 0.25
    if not isinstance(kind, float):
        x[1::2, 1] = torch.randn(G // 2, V, device=dev, generator=g) * 4
    x = x.to(dtype)
    d = x.double()
    lse = torch.logsumexp(d, 2)
    best = d.amax(2) - lse
    gap = torch.logspace(-24, -16, G // 4, base=2, device=dev, dtype=torch.float64).repeat_interleave(4) * torch.tensor([1.0, 1.0, -1.0, -1.0], device=dev, dtype=torch.float64).repeat(G // 4)
    # the sum of the beam whose score has the finer steps is put beside the other's
    scores = torch.empty(G, B, device=dev)
    scores[:, 0] = (-0.06 - best[:, 0]).float()
    scores[:, 1] = (scores[:, 0].double() + best[:, 0] + gap - best[:, 1]).float()
    top, token = torch.sort(d, dim=2, descending=True, stable=True)
    value = (scores.double()[:, :, None] + (top[:, :, :keep] - lse[:, :, None])).reshape(G, B * keep)
    order = torch.sort(value, dim=1, descending=True, stable=True).indices[:, :keep]
    token = torch.gather(token[:, :, :keep].reshape(G, B * keep), 1, order)
    ahead = value.reshape(G, B, keep)[:, 0, 0] > value.reshape(G, B, keep)[:, 1, 0]
    assert 0.3 < ahead.float().mean() < 0.7
    s, p, t = ops.beam_candidates(x.reshape(G * B, V), scores, keep)
    assert torch.equal(p.long(), order // keep) and torch.equal(t.long(), token), (int((p.long() != order // keep).sum()), int((t.long() != token).sum()))
    want = torch.gather(value, 1, order).cpu().numpy()
    assert (np.abs(s.cpu().numpy() - want) <= SCORE(want)).all()
    # kept one: what is cut lies as close
    s1, p1, t1 = ops.beam_candidates(x.reshape(G * B, V), scores, 1)
    assert torch.equal(p1, p[:, :1]) and torch.equal(t1, t[:, :1]) and torch.equal(s1, s[:, :1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [700, 32001, 152064])
def test_beams_closer_than_float32_numbers_are(V, dtype):
    """A row of many logits beside one of a single logit, whose continuations' scores are near 0 and 2^-40 to 2^-24 apart: what tells them apart is the first row's sum.  Sums of at most 152,064
    float64 exponentials, each right to 2^-51, added in some hundreds of steps a thread: within 2^-42 of the float64 reference, with room."""
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    G = 136
    g = torch.Generator(device=dev).manual_seed(V + 1)
    x = torch.full((G, 2, V), -math.inf, device=dev)
    x[:, 0] = torch.randn(G, V, device=dev, generator=g) * torch.linspace(0, 9, G, device=dev)[:, None]
    x[::3, 0, ::5], x[1::3, 0, 3::7] = -math.inf, math.nan
    x[:, 1, 2] = 11.0
    x = x.to(dtype)
    d = torch.nan_to_num(x[:, 0].double(), nan=-math.inf)
    best = d.amax(1) - torch.logsumexp(d, 1)
    gap = torch.logspace(-40, -24, G // 2, base=2, device=dev, dtype=torch.float64).repeat_interleave(2) * torch.tensor([1.0, -1.0], device=dev, dtype=torch.float64).repeat(G // 2)
    scores = torch.empty(G, 2, device=dev)
    scores[:, 0] = -best.float()
    scores[:, 1] = (scores[:, 0].double() + best + gap).float()
    away = scores[:, 1].double() - (scores[:, 0].double() + best)
    assert (away.abs() > 2.0 ** -42).all()
    _, p, _ = ops.beam_candidates(x.reshape(2 * G, V), scores, 1)
    assert torch.equal(p[:, 0] == 1, away > 0), torch.nonzero((p[:, 0] == 1) != (away > 0)).tolist()


@pytest.mark.parametrize("keep", [1, 7, 64, 128])
@pytest.mark.parametrize("kind", ["rising", "falling", "level", "steps"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_candidates_of_long_whole_rows(keep, kind, dtype):
    """More rows than the SMs hold blocks, so that each is read whole by one block, in all its runs: logits that rise through the row (every run finds more than its lists hold),
    fall, are equal (the first tokens win), or rise in steps."""
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    G, B, V = 20, 31, 100003 if kind == "rising" else 100000
    at = torch.arange(V, device=dev, dtype=torch.float64)
    row = {"rising": at * 1e-4, "falling": -at * 1e-4, "level": at * 0 - 3.0, "steps": (at // 5000)}[kind].to(dtype)
    logits = row[None].expand(G * B, V).contiguous()
    scores = -torch.rand(G, B, device=dev, generator=torch.Generator(device=dev).manual_seed(keep)) * 1e-3
    s, p, t = ops.beam_candidates(logits, scores, keep)
    x = row.double()
    best = torch.sort(x, descending=True, stable=True).indices[:keep]
    lp = torch.log_softmax(x, 0)[best]
    # all beams' rows are the same: s differs by the scores alone
    value = (scores.double()[:, :, None] + lp[None, None]).reshape(G, B * keep)
    order = torch.sort(value, dim=1, descending=True, stable=True).indices[:, :keep]
    assert torch.equal(p.long(), order // keep) and torch.equal(t.long(), best[order % keep])
    want = torch.gather(value, 1, order).cpu().numpy()
    # (25 batches a thread in place of the 19 that SCORE counts: 6 additions more)
    assert (np.abs(s.cpu().numpy() - want) <= SCORE(want) + 6 * 2.0 ** -24).all()


def test_candidates_of_no_search():
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    s, p, t = ops.beam_candidates(torch.empty(0, 50, device=dev), torch.empty(0, 4, device=dev), 8)
    assert s.shape == p.shape == t.shape == (0, 8)


def _random_step(rng, G, B, K, stops, full):
    stop = list(range(1, 1 + stops))
    s = -np.sort(rng.uniform(1, 9, (G, K)).astype(np.float32).round(2), axis=1)          # (ties among them)
    p, t = rng.integers(0, B, (G, K)), rng.integers(5, 50, (G, K))
    if stops:
        at = rng.random((G, K)) < 0.4
        t[at] = rng.choice(stop, at.sum())
    short = rng.random(G) < 0.3
    for g in np.flatnonzero(short):
        n = rng.integers(0, K + 1)
        s[g, n:], p[g, n:], t[g, n:] = -np.inf, -1, -1
    W = int(rng.integers(1, 33)) if B > 1 else 1
    pool = []
    for g in range(G):
        n = W if full else int(rng.integers(0, W + 1))
        held = -np.sort(rng.uniform(0.1, 3, n).astype(np.float32).round(2))
        pool.append([(v, int(rng.integers(1, 9)), int(rng.integers(0, B)), int(rng.integers(1, 50))) for v in held])
    return s, p, t, stop, W, pool, rng.integers(0, 12, G), (rng.random(G) < 0.15).astype(int)


@pytest.mark.parametrize("B,K", [(1, 1), (1, 3), (4, 8), (7, 40), (32, 128), (20, 5)])
@pytest.mark.parametrize("stops", [0, 1, 3])
@pytest.mark.parametrize("power", [0.0, 1.0, 0.7, -0.5])
def test_advance(B, K, stops, power):
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    for full in (False, True):
        rng = np.random.default_rng(B * 100 + K + stops)
        G, max_new = 33, 11
        s, p, t, stop, W, pool, lengths, done = _random_step(rng, G, B, K, stops, full)
        flat = [np.array([[e[i] for e in r] + [[-np.inf, 3, 3, 3][i]] * (W - len(r)) for r in pool]) for i in range(4)]
        held = ops.BeamPool(torch.tensor(flat[0], dtype=torch.float32, device=dev), *(_i32(f, dev) for f in flat[1:]))
        args = (torch.tensor(s, device=dev), _i32(p, dev), _i32(t, dev))
        kw = dict(beams=B, stop_ids=_i32(stop, dev) if stops else None, max_new=max_new, length_penalty=power)
        got = ops.beam_advance(*args, held, _i32(lengths, dev), _i32(done, dev), **kw)
        # the same into the inputs' own tensors
        n2, d2 = _i32(lengths, dev), _i32(done, dev)
        own = ops.BeamPool(*(x.clone() for x in held))
        again = ops.beam_advance(*args, own, n2, d2, out=ops.BeamStep(None, None, None, n2, d2, own), **kw)
        assert again.pool.scores.data_ptr() == own.scores.data_ptr() and again.done.data_ptr() == d2.data_ptr()
        for a, b in zip((*got[:5], *got.pool), (*again[:5], *again.pool)):
            assert torch.equal(a, b)
        for g in range(G):
            nxt, after, n, over = plain.advance(list(zip(s[g], p[g].tolist(), t[g].tolist())), pool[g], int(lengths[g]), int(done[g]), beams=B, stop_ids=stop,
                                                max_new=max_new, power=power, width=W, seen=got.pool.scores[g].cpu().numpy())
            after = after + [(-np.inf, 0, 0, 0)] * (W - len(after))
            for i, x in enumerate(got[:3]):
                assert x[g].tolist() == [float(e[i]) if i == 0 else e[i] for e in nxt], (g, i)
            assert (int(got.lengths[g]), int(got.done[g])) == (n, over)
            assert got.pool.scores[g].tolist() == [float(e[0]) for e in after]
            for i in (1, 2, 3):
                assert got.pool[i][g].tolist() == [e[i] for e in after]


@pytest.mark.parametrize("power,max_new", [(-6.4, 1000), (6.4, 1000), (-16.0, 16), (63.0, 2), (-2.1, 1 << 29), (-1.0, 100)])
def test_advance_at_the_ends_of_float32(power, max_new):
    """Penalties up to the largest that are taken, scores from one step of float32 below 0 to its lowest number: nothing that finishes is lost, and the pool is in the order of the scores."""
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    low = float(torch.finfo(torch.float32).min)
    s = torch.tensor([[-(2.0 ** -24), -1.0, -50.0, -1e12, -1e30, low]], device=dev)
    got = ops.beam_advance(s, _i32([[0, 1, 2, 3, 4, 5]], dev), _i32([[9, 8, 7, 6, 5, 4]], dev), ops.beam_pool(1, 6, dev), _i32([max_new - 1], dev), _i32([0], dev), beams=6, max_new=max_new,
                           length_penalty=power)
    exact = s[0].double().cpu().numpy() / np.float64(max_new) ** power
    want = np.maximum(exact, np.float64(low))
    pool = got.pool.scores[0].cpu().numpy().astype(np.float64)
    assert (np.abs(pool - want) <= 2.0 ** -24 * np.abs(want)).all(), (pool, want)
    assert got.pool.tokens[0].tolist() == [9, 8, 7, 6, 5, 4] and got.pool.lengths[0].tolist() == [max_new] * 6 and got.done.tolist() == [1]


def _reorder_case(rng, G, B, lens, stride_of, kinds, dev):
    """Pages of every search: shared whole ones, then one a beam and column; states of several types."""
    paged = []
    for (outer, heads, ps, hd, dtype), stride in zip(kinds, stride_of):
        entries = np.asarray(lens) // stride
        shared = entries // ps
        columns = int(shared.max()) + 3
        pages = int(shared.sum() + G * B * 3 + 4)
        ids = list(rng.permutation(pages))
        table = np.full((G * B, columns), -1)
        for g in range(G):
            common = [ids.pop() for _ in range(shared[g])]
            for b in range(B):
                table[g * B + b, :shared[g]] = common
                table[g * B + b, shared[g]:shared[g] + 3] = [ids.pop() for _ in range(3)]
        storage = torch.tensor(rng.integers(-120, 120, outer + (pages, heads, ps, hd)), device=dev).to(dtype)
        paged.append((storage, table, stride))
    return paged


@pytest.mark.parametrize("G,B", [(1, 1), (1, 2), (3, 4), (5, 7), (2, 32), (64, 32)])
@pytest.mark.parametrize("dup", [0.0, 0.5, 1.0])
def test_reorder(G, B, dup):
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    rng = np.random.default_rng(G * 100 + B + int(10 * dup))
    many = G * B > 500
    lens = rng.integers(0, 40 if many else 200, G)
    lens[0] = 32                                        # whole pages only
    kinds = [((3, 2), 2, 16, 64, torch.bfloat16), ((2, 1), 1, 8, 20, torch.float32), ((1, 2), 3, 16, 3, torch.bfloat16)]
    paged = _reorder_case(rng, G, B, lens, (1, 4, 1), kinds, dev)
    parents = np.stack([rng.permutation(B) for _ in range(G)])
    again = rng.random((G, B)) < dup
    parents[again] = rng.integers(-1 if dup < 1 else 0, B, again.sum())
    if dup == 1.0:
        parents[0] = 0
    rows = G * B + 1
    slots = rng.permutation(rows)[:G * B]
    states = [torch.randn(rows, 5, 8, 8, device=dev), torch.randn(rows, 3, device=dev), torch.randint(0, 250, (rows, 37), device=dev).to(torch.uint8),
              torch.randn(rows, 1, device=dev), torch.randn(rows, 40 if many else 9000, device=dev).to(torch.bfloat16)]
    want_states = [s.clone().cpu().view(torch.int16).numpy() if s.dtype == torch.bfloat16 else s.clone().cpu().numpy() for s in states]
    want_paged = [((s.clone().cpu().view(torch.int16) if s.dtype == torch.bfloat16 else s.clone().cpu()).numpy(), t.copy(), st) for s, t, st in paged]
    want_slots, want_tables = plain.reorder(parents, slots, lens, want_states, want_paged)
    slots_d, tables_d = _i32(slots, dev), [_i32(t, dev) for _, t, _ in paged]
    got_slots, got_tables = ops.beam_reorder(_i32(parents, dev), slots_d, _i32(lens, dev), states=states, paged=[(s, t, st) for (s, _, st), t in zip(paged, tables_d)])
    assert np.array_equal(got_slots.cpu().numpy(), want_slots)
    assert np.array_equal(slots_d.cpu().numpy(), slots)
    for a, b in zip(got_tables, want_tables):
        assert np.array_equal(a.cpu().numpy(), b)
    for s, w in zip(states, want_states):
        assert np.array_equal((s.cpu().view(torch.int16) if s.dtype == torch.bfloat16 else s.cpu()).numpy(), w)
    for (s, _, _), (w, _, _) in zip(paged, want_paged):
        assert np.array_equal((s.cpu().view(torch.int16) if s.dtype == torch.bfloat16 else s.cpu()).numpy(), w)


def test_reorder_of_more_states_and_caches_than_a_launch_takes():
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    rng = np.random.default_rng(3)
    G, B, lens = 2, 3, [21, 5]
    paged = _reorder_case(rng, G, B, lens, (1,) * 11, [((1, 2), 1, 16, 8, torch.float32)] * 11, dev)
    parents, slots = np.array([[1, 1, 0], [2, 2, 2]]), np.array([4, 2, 0, 1, 3, 5])
    states = [torch.randn(7, 4 + i % 3, device=dev) for i in range(130)]
    want_states = [s.cpu().numpy().copy() for s in states]
    want_paged = [(s.cpu().numpy().copy(), t.copy(), st) for s, t, st in paged]
    want_slots, want_tables = plain.reorder(parents, slots, lens, want_states, want_paged)
    got_slots, got_tables = ops.beam_reorder(_i32(parents, dev), _i32(slots, dev), _i32(lens, dev), states=states, paged=[(s, _i32(t, dev), st) for s, t, st in paged])
    assert np.array_equal(got_slots.cpu().numpy(), want_slots)
    assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(got_tables, want_tables))
    assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(states, want_states))
    assert all(np.array_equal(s.cpu().numpy(), w) for (s, _, _), (w, _, _) in zip(paged, want_paged))


def test_reorder_leaves_alone_what_tables_do_not_name():
    """Slots and pages outside their storage, negative ones, a context behind the table: nothing is copied there, the rest is."""
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    kv = torch.randn(1, 2, 4, 1, 16, 8, device=dev)
    before = kv.clone()
    state = torch.randn(3, 4, device=dev)
    held = state.clone()
    table = _i32([[0, -1], [1, 99]], dev)
    slots, tables = ops.beam_reorder(_i32([[0, 0]], dev), _i32([0, 7], dev), _i32([20], dev), states=[state], paged=[(kv, table, 1)])
    assert torch.equal(kv, before) and torch.equal(state, held) and slots.tolist() == [0, 7] and tables[0].tolist() == [[0, -1], [0, 99]]
    _, tables = ops.beam_reorder(_i32([[1, 1]], dev), _i32([0, 1], dev), _i32([500], dev), states=[state], paged=[(kv, table, 1)])
    assert torch.equal(kv, before) and torch.equal(state[0], held[1]) and tables[0].tolist() == [[1, 99], [1, 99]]


def test_reorder_beyond_four_gigabytes():
    """Rows of state and pages whose offsets pass 32 bits."""
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    n = 2_500_000_016
    state = torch.empty(3, n, dtype=torch.uint8, device=dev)
    for i in range(3):
        state[i].fill_(7 + i)
    kv = torch.zeros(2, 2, 70_000, 1, 16, 512, dtype=torch.bfloat16, device=dev)           # 4.6 GB
    kv[:, :, 5], kv[:, :, 69_999] = 3.0, 1.0
    # beam 2 has no child: beam 1 becomes a second child of beam 0 in beam 2's places
    slots, tables = ops.beam_reorder(_i32([[0, 0, 1]], dev), _i32([0, 1, 2], dev), _i32([9], dev), states=[state], paged=[(kv, _i32([[5], [6], [69_999]], dev), 1)])
    assert slots.tolist() == [0, 2, 1] and tables[0].tolist() == [[5], [69_999], [6]]
    for row, value in ((0, 7), (1, 8), (2, 7)):
        assert int(state[row].min()) == int(state[row].max()) == value
    assert (kv[:, :, 69_999, :, :9] == 3).all() and (kv[:, :, 69_999, :, 9:] == 1).all() and (kv[:, :, 5] == 3).all() and not kv[:, :, 6].any()
    del state, kv
    torch.cuda.empty_cache()


@pytest.mark.parametrize("S,most", [(1, 1), (1, 700), (5, 1), (48, 40), (300, 9), (1100, 2)])
@pytest.mark.parametrize("grow", [False, True])
@pytest.mark.parametrize("ps,strides", [(16, (1,)), (8, (1, 4)), (5, (1, 7, 3))])
def test_step_tables(S, most, grow, ps, strides):
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    rng = np.random.default_rng(S + most + ps)
    q = rng.integers(0 if S > 1 else 1, most + 1, S)
    have = np.where(rng.random(S) < 0.2, 0, rng.integers(0, 500, S))
    rows = rng.permutation(S + 2)[:S]
    tables, free = [], []
    for st in strides:
        had, needs = -(-(have // st) // ps), -(-((have + q) // st) // ps)
        columns = int(needs.max()) + (1 if st == 1 else 4)
        ids = rng.permutation(int(needs.sum()) + 9)
        held = had if grow else needs
        table, at = np.full((S + 2, columns), -1), 0
        for s in range(S):
            table[rows[s], :held[s]] = ids[at:at + held[s]]
            at += held[s]
        tables.append(table)
        free.append(ids[at:] if grow else None)
    if S > 1:
        tables[0][rows[0], 0] = -1                        # a page given back by a window
    for T in sorted({int(q.sum()), int(q.sum()) + 13, max(0, int(q.sum()) - 3)}):
        columns = [t.shape[1] + (2 if k else 0) for k, t in enumerate(tables)]
        want_tables = [t.copy() for t in tables]
        want = plain.step_tables(q, have, want_tables, page_size=ps, num_tokens=T, strides=strides, rows=rows, free=free, columns=columns)
        dev_tables = [_i32(t, dev) for t in tables]
        got = ops.step_tables(_i32(q, dev), _i32(have, dev), dev_tables, page_size=ps, num_tokens=T, strides=strides, rows=_i32(rows, dev),
                              free=[_i32(f, dev) if f is not None else None for f in free], columns=columns)
        for a, b in zip((*got[:4], *got.block_tables, *got.slot_mappings, *dev_tables), (*want[:4], *want[4], *want[5], *want_tables)):
            assert np.array_equal(a.cpu().numpy(), b)


def test_step_tables_with_too_few_free_pages_and_columns():
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    q, have = [40, 3, 30], [5, 16, 0]
    tables = [[[7, -1, -1], [8, -1, -1], [-1, -1, -1]]]
    free = [[3, 4, 5, 6]]                                 # 2 + 1 + 2 are wanted
    want_t = [np.array(t) for t in tables]
    want = plain.step_tables(np.array(q), np.array(have), want_t, page_size=16, num_tokens=73, strides=[1], rows=np.arange(3), free=[np.array(free[0])], columns=[2])
    t = _i32(tables[0], dev)
    got = ops.step_tables(_i32(q, dev), _i32(have, dev), [t], page_size=16, num_tokens=73, free=[_i32(free[0], dev)], columns=[2])
    for a, b in zip((*got[:4], *got.block_tables, *got.slot_mappings, t), (*want[:4], *want[4], *want[5], *want_t)):
        assert np.array_equal(a.cpu().numpy(), b)
    none = ops.step_tables(_i32([2], dev), _i32([0], dev), [t], page_size=16, num_tokens=2, rows=_i32([9], dev))         # a row that there is not
    assert none.slot_mappings[0].tolist() == [-1, -1] and none.block_tables[0].tolist() == [[-1] * 3]
    empty = ops.step_tables(_i32([2], dev), _i32([0], dev), [t], page_size=16, num_tokens=2, rows=_i32([2], dev), free=[_i32([], dev)])
    assert empty.slot_mappings[0].tolist() == [-1, -1] and t[2].tolist() == [-1, -1, -1]


def test_one_step_captured_and_replayed_on_another_stream():
    """Candidates, advance, reorder and tables as one graph: replays give what the calls gave, with the graph's inputs changed in between."""
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    G, B, V, ps = 3, 4, 5003, 16
    logits, scores = torch.empty(G * B, V, device=dev), torch.empty(G, B, device=dev)
    lengths, done, lens = _i32([3] * G, dev), _i32([0] * G, dev), _i32([37, 20, 64], dev)
    slots, table = _i32(np.arange(G * B), dev), _i32(np.arange(G * B * 6).reshape(G * B, 6), dev)
    kv, state = torch.empty(2, 2, G * B * 6, 2, ps, 64, device=dev, dtype=torch.bfloat16), torch.empty(G * B, 1000, device=dev)
    pool, stop = ops.beam_pool(G, B, dev), _i32([17, 900], dev)

    def fill(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        logits.copy_(torch.randn(G * B, V, device=dev, generator=g) * 3)
        scores.copy_(-torch.rand(G, B, device=dev, generator=g) * 3)
        kv.copy_(torch.randn(kv.shape, device=dev, generator=g))
        state.copy_(torch.randn(state.shape, device=dev, generator=g))

    def step():
        c = ops.beam_candidates(logits, scores, 12)
        nxt = ops.beam_advance(*c, pool, lengths, done, beams=B, stop_ids=stop, max_new=20)
        new_slots, tables = ops.beam_reorder(nxt.parents, slots, lens, states=[state], paged=[(kv, table, 1)])
        have = lens[:, None].expand(G, B).reshape(-1).contiguous()
        t = ops.step_tables(torch.ones_like(have), have, tables, page_size=ps, num_tokens=G * B)
        return (*c, *nxt[:5], *nxt.pool, new_slots, *tables, *t[:4], *t.block_tables, *t.slot_mappings, kv.clone(), state.clone())
    fill(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    side = torch.cuda.Stream()
    for seed in (1, 2):
        fill(seed)
        want = [x.clone() for x in step()]
        fill(seed)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(held, want):
            assert torch.equal(a, b)


def test_two_streams_at_once_and_the_same_bits_every_time():
    """Calls on two streams side by side have scratch of their own; lists that fill in any order give one result."""
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    g = torch.Generator(device=dev).manual_seed(11)
    sets = [(torch.randn(6 * 4, 50021, device=dev, generator=g) * 3, -torch.rand(6, 4, device=dev, generator=g)) for _ in range(2)]
    want = [ops.beam_candidates(x, s, 24) for x, s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(20):
        for (x, s), stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(ops.beam_candidates(x, s, 24))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(r, want[i % 2]))


@pytest.mark.parametrize("written", [False, True], ids=["tables", "tables-write"])
@pytest.mark.parametrize("form", ["tma", "mma", "simt"])
@pytest.mark.parametrize("source", ["tables", "reorder"])
def test_attention_right_behind_the_operators_that_make_its_tables(form, written, source):
    """Attention reads lengths and block tables before it waits for the kernel before; what `step_tables` and `beam_reorder` made is there all the same, launch by launch and in a graph.  The tensors
    written are the same ones every turn, so that what lay there before would be another turn's pages."""
    import sllm_b200.ops as ops
    dev = cuda_or_skip()
    S, nq, nkv, hd, ps, columns = 4, 8, 2, 128, 16, 12
    pages = 3 * S * columns
    g = torch.Generator(device=dev).manual_seed(2)
    kv0 = torch.randn(2, pages, nkv, ps, hd, device=dev, generator=g).bfloat16()
    kv = kv0.clone()
    qkv = torch.randn(S, (nq + 2 * nkv) * hd, device=dev, generator=g).bfloat16()
    q = qkv[:, :nq * hd].contiguous()
    rng = np.random.default_rng(2)
    sets = [(_i32(rng.permutation(pages)[:S * columns].reshape(S, columns), dev), _i32(rng.integers(1, ps * columns - 2, 2).repeat(2), dev), _i32([rng.permutation(2).tolist() for _ in range(2)], dev))
            for _ in range(6)]
    q_lens, slots = _i32([1] * S, dev), _i32(range(S), dev)
    now = [x.clone() for x in sets[0]]
    empty = lambda *n: torch.zeros(n, dtype=torch.int32, device=dev)                                 # noqa: E731
    out = ops.StepTables(empty(S + 1), empty(S), empty(S), empty(S), (empty(S, columns),), (empty(S),))
    mine = (empty(S), [empty(S, columns)])
    tiles, _ = ops.attention_tiles([1] * S, nq // nkv, dev)
    result = torch.empty_like(q)

    def turn(wait):
        t = ops.step_tables(q_lens, now[1], [now[0]], page_size=ps, num_tokens=S, out=out)
        wait()
        bt = t.block_tables[0]
        if source == "reorder":
            bt = ops.beam_reorder(now[2], slots, t.ctx_len, paged=[(kv, bt, 1)], out=mine)[1][0]
            wait()
        if written:
            ops.rope_kv_write(qkv, None, t.positions, None, 0, nq, nkv, hd, t.slot_mappings[0], kv[0], kv[1], torch.bfloat16)
            wait()
        if form == "simt":
            result.copy_(ops.attention_simt(q, kv[0], kv[1], bt, t.positions, t.seq_of_token, nq, nkv, hd, 0.1, None).view(S, -1))
        elif form == "mma":
            ops.attention_mma(q, kv[0], kv[1], bt, t.q_start, t.ctx_len, tiles, True, 1, nq, nkv, hd, 0.1, None, result)
        else:
            ops.attention_tma_decode(q, kv[0], kv[1], bt, t.q_start, t.ctx_len, tiles, 2, nq, nkv, hd, 0.1, None, result)

    def take(i):
        for a, b in zip(now, sets[i]):
            a.copy_(b)
        kv.copy_(kv0)
        result.fill_(7.0)
    want = []
    for i in range(len(sets)):
        take(i)
        torch.cuda.synchronize()
        turn(torch.cuda.synchronize)
        torch.cuda.synchronize()
        want.append(result.clone())
    assert all(not torch.equal(a, b) for a, b in itertools.combinations(want, 2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turn(lambda: None)
    for step in (lambda: turn(lambda: None), graph.replay):
        for i in list(range(len(sets))) * 5:
            take(i)
            step()
            assert torch.equal(result, want[i]), i
    ops.check_tcgen05_status()
