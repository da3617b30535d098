"""Beam search through the engine, for every architecture: against a search over the plain implementation's logits, on the CPU with the operators' plain statements in the kernels'
place and on the GPU (marked gpu) with the kernels, from captured graphs and without.  And what the cache manager, the operators' checks and the command line have to
keep."""

import itertools

import numpy as np
import pytest
import torch

from sllm_b200.cache.manager import CacheManager
from sllm_b200.cache.pools import OutOfPages
from sllm_b200.parts.base import PagedKV, SlotState
from sllm_b200.sampling import BeamParams, SamplingParams
from tests.conftest import TINY, make_model_dir
from tests.plain import beam_plain as plain

ARCHITECTURES = ("qwen2", "rososun", "nutopel", "kidolorn", "gerupel", "sezopel", "muzulorn")


@pytest.fixture(params=[pytest.param("cpu", id="stand-in"), pytest.param("cuda:0", id="gpu", marks=pytest.mark.gpu)])
def dev(request):
    """The device a body runs on; on the CPU the PyTorch stand-ins take the kernels' place."""
    if request.param == "cpu":
        request.getfixturevalue("beam_cpu_ops")
    elif not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return request.param


@pytest.fixture
def beam_cpu_ops(cpu_ops, monkeypatch):
    for name, fn in plain.CPU_OPS.items():
        monkeypatch.setattr(cpu_ops, name, fn)
    return cpu_ops


def _model(tmp_path, arch, which="A"):
    """(folder, page size, vocabulary, logits behind a sequence of ids from the plain implementation)."""
    if arch == "qwen2":
        from tests.plain import qwen2_plain as m
        config, init, page = TINY["A"]
        d = make_model_dir(tmp_path, config, init)
    else:
        import importlib
        t = importlib.import_module(f"tests.test_{arch}")
        m = importlib.import_module(f"tests.plain.{arch}_plain")
        config, page = t.CONFIGS[which]
        d = t.make_model(tmp_path, config)
    cfg, w = m.load_model(d)
    order = {"qwen2": lambda ids: m.forward(ids, w, cfg), "gerupel": lambda ids: m.forward(cfg, w, ids)}.get(arch, lambda ids: m.forward(ids, cfg, w))
    memory = {}

    def logits_of(ids):
        key = tuple(ids)
        if key not in memory:
            memory[key] = np.asarray(order(list(ids))[-1], dtype=np.float64)
        return memory[key]
    return d, page, config.get("vocab_size", config.get("vocab")), logits_of


def _llm(d, page, dev, slots, pages, **kw):
    from sllm_b200.engine.llm import LLM
    return LLM(d, dtype=kw.pop("dtype", "float32"), device=dev, block_size=page, num_pages=pages, max_num_seqs=slots, chunk_size=24, max_batch_tokens=40, **kw)


def _check(results, want, prompt, logits_of, params, what):
    """Rank by rank the plain search's scores, and every result's score is what the plain logits give its ids.  The engine's float32 logits are within 3e-4 (1 + |logit|) of the plain ones
    (the architectures' own tests), a log-probability within twice that of its largest logit's; a score is a sum of n of them over n^p."""
    assert len(results) == len(want), (what, len(results), len(want))
    for r, (ids, norm, reason) in zip(results, want):
        n = len(r.ids) + (r.finish_reason == "stop")
        total, slack = 0.0, 0.0
        for i in range(len(r.ids)):
            logits = logits_of(list(prompt) + r.ids[:i])
            total += plain.log_softmax(logits)[r.ids[i]]
            slack += 6e-4 * (1 + np.abs(logits).max())
        if r.finish_reason == "stop":
            logits = logits_of(list(prompt) + r.ids)
            total += max(plain.log_softmax(logits)[s] for s in params.stop_ids)
            slack += 6e-4 * (1 + np.abs(logits).max())
        scale = n ** params.length_penalty
        assert abs(r.score - total / scale) <= slack / scale, (what, r, total / scale)
        assert abs(r.score - norm) <= 2 * slack / scale, (what, r, ids, norm, reason)
    assert len({tuple(r.ids) + (r.finish_reason,) for r in results}) == len(results)


@pytest.mark.parametrize("arch", ARCHITECTURES)
def test_search_of_every_architecture(tmp_path, arch, dev):
    """Two prompts side by side, one longer than a page and a portion; stop ids and lengths; from graphs and launch by launch."""
    d, page, vocab, logits_of = _model(tmp_path, arch)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, vocab, n).tolist() for n in (37, 3)]
    # stops that the search meets: the likeliest tokens behind the prompts
    stops = tuple(int(np.argmax(logits_of(p))) for p in prompts)
    cases = [BeamParams(beams=3, max_new=6), BeamParams(beams=4, max_new=7, length_penalty=0.5, stop_ids=stops[:1], results=2)]
    for params in cases:
        want = [plain.search(logits_of, p, beams=params.beams, max_new=params.max_new, stop_ids=params.stop_ids, power=params.length_penalty, width=params.results) for p in prompts]
        for graphs in ((False,) if dev == "cpu" else (True, False)):
            llm = _llm(d, page, dev, 9, 400, cuda_graphs=graphs)
            for again in range(2):                            # the second time from the buffers and the graph of the first
                got = llm.beam_search(prompts, params)
                for p, g, w in zip(prompts, got, want):
                    _check(g, w, p, logits_of, params, (arch, graphs, again, params))
            assert not llm.engine.cache.requests
            llm.engine.cache.check()
            assert all(g.pool.used_count == 0 for g in llm.engine.cache.groups)


@pytest.mark.parametrize("arch,which", [(a, "A") for a in ARCHITECTURES] + [("rososun", "only_delta"), ("nutopel", "only_gla"), ("sezopel", "retention"), ("gerupel", "odd")])
def test_search_over_page_borders_with_freed_pages_poisoned(tmp_path, arch, which, dev, monkeypatch):
    """Prompts that end at a page's border and just before it, continuations that fill pages, models without any page; pages nobody holds are full of NaN."""
    monkeypatch.setenv("SLLM_POISON_FREED_PAGES", "1")
    d, page, vocab, logits_of = _model(tmp_path, arch, which)
    rng = np.random.default_rng(7)
    prompts = [rng.integers(0, vocab, n).tolist() for n in (30, 16, 1)]
    params = BeamParams(beams=3, max_new=19, length_penalty=0.0, results=3)
    llm = _llm(d, page, dev, 9, 500)
    for p, g in zip(prompts, llm.beam_search(prompts, params)):
        _check(g, plain.search(logits_of, p, beams=3, max_new=19, power=0.0), p, logits_of, params, (arch, which, len(p)))
    llm.engine.cache.check()


@pytest.mark.parametrize("arch", ARCHITECTURES)
def test_rows_of_a_search_that_is_over_at_once_hold_its_prompt(tmp_path, arch, dev, monkeypatch):
    """A search whose likeliest first token is a stop, with one result wanted, is over before its other beams held anything.  Their rows run on beside the other search: over pages that are
    theirs or the prompt's, and over numbers (pages nobody holds are full of NaN here)."""
    import sllm_b200.ops as ops
    monkeypatch.setenv("SLLM_POISON_FREED_PAGES", "1")
    d, page, vocab, logits_of = _model(tmp_path, arch)
    rng = np.random.default_rng(12)
    prompts = [rng.integers(0, vocab, n).tolist() for n in (2 * page + 5, 7)]
    stop = int(np.argmax(logits_of(prompts[0])))
    params = BeamParams(beams=3, max_new=6, stop_ids=(stop,), results=1, length_penalty=0.0)       # (no later one can score above the best first)
    seen, logits_seen, tables_of, candidates = [], [], ops.step_tables, ops.beam_candidates

    def step_tables(q_lens, have, pages, **kw):
        made = tables_of(q_lens, have, pages, **kw)
        if not (torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()):
            seen.append([(made.ctx_len.cpu().clone(), [t.cpu().clone() for t in made.block_tables], kw["strides"], kw["page_size"])])
        return made

    def beam_candidates(logits, scores, keep):
        if logits.shape[0] > len(prompts):
            logits_seen.append(logits.float().cpu().clone())
        return candidates(logits, scores, keep)
    monkeypatch.setattr(ops, "step_tables", step_tables)
    monkeypatch.setattr(ops, "beam_candidates", beam_candidates)
    llm = _llm(d, page, dev, 6, 300, cuda_graphs=False)
    got = llm.beam_search(prompts, params)
    assert seen and logits_seen
    windows = any(g.need.window for g in llm.engine.cache.groups)
    for step, in seen:
        ctx, tables, strides, ps = step
        for table, stride in zip(tables, strides):
            for r, n in enumerate(ctx.tolist()):
                assert windows or (table[r, :-(-(n // stride) // ps)] >= 0).all(), (arch, r, n, table[r])
    for x in logits_seen:
        assert not torch.isnan(x).any(), arch
    assert got[0][0].ids == [] and got[0][0].finish_reason == "stop"
    for p, g in zip(prompts, got):
        _check(g, plain.search(logits_of, p, beams=3, max_new=6, stop_ids=(stop,), power=0.0, width=1), p, logits_of, params, (arch, len(p)))
    llm.engine.cache.check()


@pytest.mark.parametrize("arch", ARCHITECTURES)
def test_more_beams_than_first_tokens(tmp_path, arch, dev, monkeypatch):
    """Two tokens above minus infinity behind the prompt: the other beams idle for a step, over pages and states that hold the prompt, and are taken by the second step's continuations."""
    import sllm_b200.ops as ops
    monkeypatch.setenv("SLLM_POISON_FREED_PAGES", "1")
    d, page, vocab, logits_of = _model(tmp_path, arch)
    rng = np.random.default_rng(13)
    prompts = [rng.integers(0, vocab, n).tolist() for n in (page + 3, 2 * page)]
    two = [np.argsort(-logits_of(p))[3:5].tolist() for p in prompts]
    candidates, seen = ops.beam_candidates, []

    def beam_candidates(logits, scores, keep):
        if scores.shape[1] == 1:
            masked = torch.full_like(logits, -float("inf"))
            for g, t in enumerate(two):
                masked[g, t] = logits[g, t]
            logits = masked
        else:
            seen.append(bool(torch.isnan(logits).any()))
        return candidates(logits, scores, keep)
    monkeypatch.setattr(ops, "beam_candidates", beam_candidates)

    def masked_logits_of(g):
        def of(ids):
            logits = logits_of(ids)
            if len(ids) > len(prompts[g]):
                return logits
            masked = np.full_like(logits, -np.inf)
            masked[two[g]] = logits[two[g]]
            return masked
        return of
    params = BeamParams(beams=5, max_new=4)
    got = _llm(d, page, dev, 10, 400, cuda_graphs=False).beam_search(prompts, params)
    assert seen and not any(seen)
    for g, p in enumerate(prompts):
        want = plain.search(masked_logits_of(g), p, beams=5, max_new=4)
        assert {r.ids[0] for r in got[g]} <= set(two[g])
        assert len(got[g]) == len(want) == 5
        for r, (ids, norm, reason) in zip(got[g], want):
            slack = 12e-4 * 4 * (1 + max(np.abs(logits_of(p + r.ids[:i])).max() for i in range(4)))
            assert abs(r.score - norm) <= slack / 4, (r, ids, norm)


@pytest.mark.gpu
@pytest.mark.parametrize("arch", ARCHITECTURES)
def test_bfloat16_search_from_graphs_is_the_one_launch_by_launch(tmp_path, arch):
    """The same kernels in the same order: the same bits, and what comes back is ordered and scored as bfloat16 logits allow."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    d, page, vocab, _ = _model(tmp_path, arch, "B" if arch not in ("qwen2", "rososun") else "A")
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, vocab, n).tolist() for n in (50, 9, 17, 33)]
    params = BeamParams(beams=5, max_new=12, stop_ids=(int(vocab) - 1, 3), length_penalty=0.7)
    got = [_llm(d, page, "cuda:0", 20, 600, dtype="bfloat16", cuda_graphs=g).beam_search(prompts, params) for g in (True, False)]
    assert got[0] == got[1]
    for g in got[0]:
        assert 1 <= len(g) <= 5 and all(a.score >= b.score for a, b in zip(g, g[1:])) and all(np.isfinite(r.score) and len(r.ids) <= 12 for r in g)


def test_parameters_changed_between_calls(tmp_path, dev):
    """What was kept for one call's parameters is not taken for another's, though both are one object that the caller changes."""
    d, page, vocab, logits_of = _model(tmp_path, "qwen2")
    prompt = np.random.default_rng(2).integers(0, vocab, 11).tolist()
    llm = _llm(d, page, dev, 4, 60)
    params = BeamParams(beams=3, max_new=3)
    for new, beams in ((3, 3), (6, 3), (3, 3), (4, 2), (3, 3), (5, 4), (2, 1), (7, 3), (3, 3)):
        params.max_new, params.beams, params.results = new, beams, beams
        _check(llm.beam_search([prompt], params)[0], plain.search(logits_of, prompt, beams=beams, max_new=new), prompt, logits_of, params, (new, beams))
    params.beams = 40
    with pytest.raises(ValueError):
        llm.beam_search([prompt], params)


def test_search_beside_running_requests_and_one_after_another(tmp_path, dev):
    """Searches take what is free: with slots for one search they run one after another, beside a request that is being decoded, whose tokens stay what they are alone."""
    d, page, vocab, logits_of = _model(tmp_path, "qwen2")
    rng = np.random.default_rng(4)
    prompts, other = [rng.integers(0, vocab, n).tolist() for n in (18, 5, 33)], rng.integers(0, vocab, 21).tolist()
    params = BeamParams(beams=4, max_new=5)
    alone = _llm(d, page, dev, 5, 60).generate([other], SamplingParams(max_new=12))[0].ids
    llm = _llm(d, page, dev, 5, 60)
    req = llm.add_request(other, SamplingParams(max_new=12))
    for _ in range(4):
        llm.step()
    got = llm.beam_search(prompts, params)
    while req.status != "finished":
        llm.step()
    assert req.output == alone
    for p, g in zip(prompts, got):
        _check(g, plain.search(logits_of, p, beams=4, max_new=5), p, logits_of, params, "one after another")
    # more beams than tokens in the vocabulary's top at the first step, one token, one beam
    for params in (BeamParams(beams=1, max_new=4), BeamParams(beams=4, max_new=1)):
        got = llm.beam_search(prompts[:1], params)[0]
        _check(got, plain.search(logits_of, prompts[0], beams=params.beams, max_new=params.max_new), prompts[0], logits_of, params, params)
    assert llm.beam_search([], params) == []


def test_one_beam_is_greedy(tmp_path, dev):
    d, page, vocab, logits_of = _model(tmp_path, "qwen2")
    prompt = np.random.default_rng(9).integers(0, vocab, 20).tolist()
    llm = _llm(d, page, dev, 4, 40)
    greedy = llm.generate([prompt], SamplingParams(max_new=9))[0].ids
    assert llm.beam_search([prompt], BeamParams(beams=1, max_new=9))[0][0].ids == greedy


def test_refused_searches(tmp_path, beam_cpu_ops):
    d, page, vocab, _ = _model(tmp_path, "qwen2")
    llm = _llm(d, page, "cpu", 4, 8)
    for prompt, params, error in (([1], BeamParams(beams=5), OutOfPages), (list(range(100)), BeamParams(beams=4, max_new=20), OutOfPages), ([], BeamParams(), ValueError),
                                  ([vocab], BeamParams(), ValueError), ([-1], BeamParams(), ValueError), ([1] * 120, BeamParams(max_new=20), ValueError),
                                  ([1], BeamParams(stop_ids=(vocab,)), ValueError)):
        with pytest.raises(error):
            llm.beam_search([prompt], params)
        assert not llm.engine.cache.requests
    for kw in (dict(beams=0), dict(beams=33), dict(max_new=0), dict(results=0), dict(results=40), dict(length_penalty=float("nan")), dict(length_penalty=64.0),
               dict(beams=32, stop_ids=range(4))):
        with pytest.raises(ValueError):
            BeamParams(**kw)
    assert BeamParams(beams=3).results == 3 and BeamParams(beams=3, stop_ids=(4, 4, 2)).keep == 9


def test_a_prompt_that_cannot_fit_is_found_before_the_others_run(tmp_path, beam_cpu_ops):
    d, page, vocab, _ = _model(tmp_path, "qwen2")
    llm = _llm(d, page, "cpu", 4, 8)
    fits, never = [1, 2, 3], list(range(100))
    steps = llm.engine.steps_run
    for prompts in ([fits, never], [fits, fits, never, fits], [never, fits]):
        with pytest.raises(OutOfPages, match="over 100"):
            llm.beam_search(prompts, BeamParams(beams=4, max_new=20))
        assert llm.engine.steps_run == steps and not llm.engine.cache.requests
    assert len(llm.beam_search([fits, fits], BeamParams(beams=4, max_new=2))) == 2


def test_a_search_that_fails_gives_everything_back(tmp_path, beam_cpu_ops, monkeypatch):
    d, page, _, _ = _model(tmp_path, "qwen2")
    llm = _llm(d, page, "cpu", 4, 40)

    def fails(*a, **k):
        raise RuntimeError("on purpose")
    monkeypatch.setattr(beam_cpu_ops, "beam_reorder", fails)
    with pytest.raises(RuntimeError, match="on purpose"):
        llm.beam_search([[1, 2, 3]], BeamParams(beams=3, max_new=4))
    assert not llm.engine.cache.requests and all(g.pool.used_count == 0 for g in llm.engine.cache.groups)


def test_the_plain_search_is_exhaustive_when_nothing_is_pruned():
    """With a beam for every prefix the search finds the best of all sequences."""
    rng = np.random.default_rng(0)
    table = {}

    def logits_of(ids):
        return table.setdefault(tuple(ids), rng.normal(size=3) * 2)
    for power in (0.0, 1.0):
        found = []
        for n in (1, 2, 3):
            for ids in itertools.product(range(3), repeat=n):
                if 0 in ids[:-1] or (n < 3 and ids[-1] != 0):
                    continue
                s = sum(plain.log_softmax(logits_of(ids[:i]))[t] for i, t in enumerate(ids))
                found.append((s / n ** power, [t for t in ids if t != 0]))
        found.sort(key=lambda f: -f[0])
        got = plain.search(logits_of, [], beams=9, max_new=3, stop_ids=(0,), power=power, width=4)
        for (ids, norm, _), (s, want) in zip(got, found):
            assert ids == want and abs(norm - s) < 1e-5


# ---- the cache manager's forks --------------------------------------------------------------------------------------------

def test_forks_share_whole_pages_and_give_back_their_own():
    needs = [("own", (PagedKV(2, 8, None), SlotState((3,)))), ("own", PagedKV(1, 4, 20)), ("own", PagedKV(1, 4, None, stride=3, name="pooled"))]
    c = CacheManager(needs, page_size=4, num_pages=40, max_requests=5)
    c.add_request("a")
    c.reserve("a", 30)
    c.commit("a", 14)
    free = [g.pool.free_count for g in c.groups]
    want = c.fork_pages("a", 30)
    assert want == [8 - 3, 8 - 3, 3 - 1]
    f = c.fork_request("a", "b", 30)
    assert [g.pool.free_count for g in c.groups] == [a - b for a, b in zip(free, want)]
    assert [t[:3].count(-1) for t in f.tables] == [3, 3, 1] and f.num_tokens == 14 and f.slot != c.requests["a"].slot
    c.check()
    with pytest.raises(ValueError, match="fork itself"):
        c.fork_request("b", "x", 30)
    with pytest.raises(ValueError, match="cannot hold"):
        c.fork_request("a", "x", 13)
    with pytest.raises(ValueError, match="forks still read"):
        c.free_request("a")
    c.fork_request("a", "c", 16)
    before = [g.pool.free_count for g in c.groups]
    with pytest.raises(OutOfPages):
        c.fork_request("a", "d", 4000)
    assert [g.pool.free_count for g in c.groups] == before and "d" not in c.requests and c.requests["a"].forks == 2
    c.free_request("b")
    c.free_request("c")
    c.free_request("a")
    c.check()
    assert all(g.pool.used_count == 0 for g in c.groups) and c.slots.free_count == 5


# ---- what the operators refuse, before anything is launched ---------------------------------------------------------------

@pytest.fixture
def unlaunched(monkeypatch):
    """The operators with their launches recorded in place of made, and CPU tensors let through."""
    import sllm_b200.ops as ops
    calls = []
    monkeypatch.setattr(ops, "_here", lambda what, *t: None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_beam_splits", lambda *a: 2)
    monkeypatch.setattr(ops, "call", lambda name, *a: calls.append((name, a)))
    return ops, calls


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_refusals_of_the_operators(unlaunched):
    ops, calls = unlaunched
    f = torch.zeros
    pool = ops.BeamPool(f(2, 3), _i(2, 3), _i(2, 3), _i(2, 3))
    state, kv, table = f(7, 4), f(2, 5, 1, 16, 8), _i(6, 2)

    def advance(s=f(2, 4), p=_i(2, 4), t=_i(2, 4), pool=pool, n=_i(2), d=_i(2), **kw):
        return ops.beam_advance(s, p, t, pool, n, d, **{**dict(beams=3, max_new=4), **kw})

    def reorder(p=_i(2, 3), s=_i(6), n=_i(2), states=(state,), paged=((kv, table, 1),), **kw):
        return ops.beam_reorder(p, s, n, states=states, paged=paged, **kw)

    def tables(q=_i(3), h=_i(3), t=(_i(4, 2),), **kw):
        return ops.step_tables(q, h, t, **{**dict(page_size=16, num_tokens=3), **kw})
    good = [lambda: ops.beam_candidates(f(6, 9), f(2, 3), 5), lambda: ops.beam_candidates(f(6, 9).bfloat16(), f(2, 3), 128), advance, lambda: advance(stop_ids=_i(2)), reorder,
            lambda: reorder(n=_i(6)), lambda: reorder(states=(), paged=()), tables, lambda: tables(rows=_i(3), free=[_i(9)], columns=[1], strides=[3])]
    for i, g in enumerate(good):
        g()
        assert len(calls) == i + 1
    bad = [lambda: ops.beam_candidates(f(6, 9).half(), f(2, 3), 5), lambda: ops.beam_candidates(f(5, 9), f(2, 3), 5), lambda: ops.beam_candidates(f(6, 9), f(2, 3).double(), 5),
           lambda: ops.beam_candidates(f(6, 9), f(2, 3), 0), lambda: ops.beam_candidates(f(6, 9), f(2, 3), 129), lambda: ops.beam_candidates(f(66, 9), f(2, 33), 5),
           lambda: ops.beam_candidates(f(6, 0), f(2, 3), 5), lambda: ops.beam_candidates(f(6, 9), f(6), 5),
           lambda: advance(s=f(2, 4).double()), lambda: advance(p=_i(2, 5)), lambda: advance(t=_i(2, 4).long()), lambda: advance(n=_i(3)), lambda: advance(d=f(2)), lambda: advance(beams=0),
           lambda: advance(beams=33), lambda: advance(max_new=0), lambda: advance(length_penalty=float("nan")), lambda: advance(length_penalty=float("inf")), lambda: advance(stop_ids=_i(2).long()),
           lambda: advance(pool=ops.BeamPool(f(2, 33), _i(2, 33), _i(2, 33), _i(2, 33))), lambda: advance(pool=pool._replace(tokens=_i(2, 4))),
           lambda: advance(out=ops.BeamStep(f(2, 4), None, None, None, None, ops.BeamPool(None, None, None, None))),
           lambda: reorder(p=_i(6)), lambda: reorder(p=_i(2, 33), s=_i(66)), lambda: reorder(s=_i(5)), lambda: reorder(n=_i(3)), lambda: reorder(p=_i(2, 3).long()),
           lambda: reorder(paged=((kv, _i(5, 2), 1),)), lambda: reorder(paged=((kv, table, 0),)), lambda: reorder(paged=((kv[0, 0], table, 1),)), lambda: reorder(paged=((kv[:0], table, 1),)),
           lambda: reorder(paged=((kv.to(torch.uint8), table, 1),)), lambda: reorder(out=(_i(6), [])), lambda: reorder(out=(_i(6), [table])), lambda: reorder(p=_i(100, 32), s=_i(3200), n=_i(100), paged=()),
           lambda: tables(q=_i(0), h=_i(0)), lambda: tables(h=_i(2)), lambda: tables(t=(_i(2, 2),)), lambda: tables(t=(_i(4, 2).long(),)), lambda: tables(page_size=0), lambda: tables(num_tokens=-1),
           lambda: tables(strides=[0]), lambda: tables(strides=[1, 1]), lambda: tables(free=[_i(2, 2)]), lambda: tables(rows=_i(2)), lambda: tables(t=(_i(4, 2),) * 9), lambda: tables(columns=[-1]),
           lambda: tables(t=(_i(4, 2), _i(5, 2)))]
    for i, b in enumerate(bad):
        with pytest.raises(ops.KernelError):
            b()
        assert len(calls) == len(good), i


def test_results_that_lie_over_what_is_read_are_refused(unlaunched):
    """Blocks of other searches, or other threads, read there while one writes."""
    ops, calls = unlaunched
    G, B, keep, W = 2, 3, 6, 3
    flat, ints = torch.zeros(400), _i(4000)
    s, p, t, lengths, done, stops = flat[:G * keep].view(G, keep), ints[:12].view(G, keep), ints[12:24].view(G, keep), ints[30:32], ints[32:34], ints[40:42]
    pool = ops.BeamPool(flat[20:26].view(G, W), *(ints[50 + 6 * i:56 + 6 * i].view(G, W) for i in range(3)))
    none = ops.BeamStep(*(None,) * 5, ops.BeamPool(*(None,) * 4))

    def advance(s=s, p=p, t=t, **out):
        held = {k: out.pop(k) for k in ("pool",) if k in out}
        ops.beam_advance(s, p, t, pool, lengths, done, beams=B, max_new=9, stop_ids=stops, out=none._replace(**out, **held))
    # a result that is the input of its kind; candidates as many as beams among them
    s3, p3, t3 = flat[100:106].view(G, B), ints[100:106].view(G, B), ints[106:112].view(G, B)
    good = [lambda: advance(pool=pool, lengths=lengths, done=done), lambda: advance(s=s3, p=p3, t=t3, scores=s3, parents=p3, tokens=t3), lambda: advance(scores=flat[12:18].view(G, B)),
            lambda: advance(pool=pool._replace(tokens=None))]
    bad = [lambda: advance(scores=flat[:6].view(G, B)), lambda: advance(scores=flat[8:14].view(G, B)), lambda: advance(parents=ints[:6].view(G, B)), lambda: advance(tokens=ints[18:24].view(G, B)),
           lambda: advance(lengths=done), lambda: advance(lengths=done, done=lengths), lambda: advance(done=stops), lambda: advance(parents=ints[200:206].view(G, B), tokens=ints[203:209].view(G, B)),
           lambda: advance(pool=pool._replace(tokens=pool.parents)), lambda: advance(pool=pool._replace(parents=pool.tokens, tokens=pool.parents)), lambda: advance(pool=pool._replace(scores=flat[23:29].view(G, W))),
           lambda: advance(s=s3, p=p3, t=t3, parents=t3), lambda: advance(s=s3, p=p3, t=t3, scores=flat[101:107].view(G, B))]
    table, other, slots, lens, kv = ints[300:312].view(6, 2), ints[400:412].view(6, 2), ints[320:326], ints[330:332], torch.zeros(2, 5, 1, 16, 8)

    def reorder(new_slots, new_table, more=()):
        ops.beam_reorder(ints[340:346].view(G, B), slots, lens, paged=((kv, table, 1), *(((kv, other, 1),) if more else ())), out=(new_slots, [new_table, *more]))
    good += [lambda: reorder(ints[500:506], ints[510:522].view(6, 2)), lambda: reorder(ints[500:506], ints[510:522].view(6, 2), (ints[522:534].view(6, 2),))]
    bad += [lambda: reorder(ints[322:328], ints[510:522].view(6, 2)), lambda: reorder(ints[500:506], ints[306:318].view(6, 2)), lambda: reorder(ints[500:506], ints[500:512].view(6, 2)),
            lambda: reorder(ints[341:347], ints[510:522].view(6, 2)), lambda: reorder(ints[327:333], ints[510:522].view(6, 2)), lambda: reorder(ints[500:506], ints[510:522].view(6, 2), (ints[410:422].view(6, 2),)),
            lambda: reorder(ints[500:506], ints[510:522].view(6, 2), (ints[521:533].view(6, 2),))]

    def tables(pages=(ints[600:608].view(4, 2),), free=None, q=ints[620:623], have=ints[630:633], slot=ints[1100:1103], **out):
        made = ops.StepTables(ints[1000:1004], ints[1010:1013], ints[1020:1023], ints[1030:1033], tuple(ints[1040 + 10 * i:1046 + 10 * i].view(3, 2) for i in range(len(pages))),
                              (slot, *(ints[1110 + 10 * i:1113 + 10 * i] for i in range(len(pages) - 1))))
        ops.step_tables(q, have, pages, page_size=16, num_tokens=3, free=free, out=made._replace(**out))
    two = (ints[600:608].view(4, 2), ints[610:618].view(4, 2))
    good += [tables, lambda: tables(pages=two, free=[ints[700:705], None]), lambda: tables(pages=(two[0], two[0])), lambda: tables(pages=two, free=[ints[700:705], ints[700:705]])]
    bad += [lambda: tables(ctx_len=ints[630:633]), lambda: tables(ctx_len=ints[628:631]), lambda: tables(q_start=ints[619:623]), lambda: tables(positions=ints[1030:1033]), lambda: tables(slot=ints[607:610]),
            lambda: tables(pages=(two[0], two[0]), free=[ints[700:705], ints[710:715]]), lambda: tables(pages=(two[0], ints[604:612].view(4, 2)), free=[ints[700:705], None]),
            lambda: tables(free=[ints[605:609]]), lambda: tables(free=[ints[700:705]], slot=ints[704:707])]
    for i, g in enumerate(good):
        g()
        assert len(calls) == i + 1, i
    for i, b in enumerate(bad):
        with pytest.raises(ops.KernelError, match="cannot be what is read"):
            b()
        assert len(calls) == len(good), i


def test_penalties_that_leave_float32_are_refused(unlaunched):
    """At 16 tokens and -33 a finished continuation's score was minus infinity, which is an empty place of the pool."""
    ops, calls = unlaunched
    pool = ops.BeamPool(torch.zeros(2, 3), _i(2, 3), _i(2, 3), _i(2, 3))
    for power, max_new, taken in ((-33.0, 16, False), (33.0, 16, False), (16.0, 16, True), (-16.0, 16, True), (16.1, 16, False), (63.0, 2, True), (63.9, 1, True), (-3.0, 1 << 29, False), (-2.1, 1 << 29, True)):
        n = len(calls)
        kw = dict(max_new=max_new, length_penalty=power)
        if taken:
            ops.beam_advance(torch.zeros(2, 4), _i(2, 4), _i(2, 4), pool, _i(2), _i(2), beams=3, **kw)
            assert len(calls) == n + 1 and BeamParams(**kw).length_penalty == power
        else:
            with pytest.raises(ops.KernelError, match="float32"):
                ops.beam_advance(torch.zeros(2, 4), _i(2, 4), _i(2, 4), pool, _i(2), _i(2), beams=3, **kw)
            with pytest.raises(ValueError, match="float32"):
                BeamParams(**kw)
            assert len(calls) == n


def test_the_operators_take_no_cpu_tensors_and_no_strided_ones():
    import sllm_b200.ops as ops
    with pytest.raises(ops.KernelError, match="CUDA device"):
        ops.beam_candidates(torch.zeros(4, 9), torch.zeros(1, 4), 4)
    with pytest.raises(ops.KernelError, match="CUDA device"):
        ops.step_tables(_i(2), _i(2), [_i(2, 3)], page_size=4, num_tokens=2)


@pytest.mark.gpu
def test_the_operators_take_no_strided_tensors_and_none_of_another_device():
    import sllm_b200.ops as ops
    from tests.conftest import cuda_or_skip
    dev = cuda_or_skip()
    with pytest.raises(ops.KernelError, match="contiguous"):
        ops.beam_candidates(torch.zeros(4, 18, device=dev)[:, ::2], torch.zeros(1, 4, device=dev), 4)
    with pytest.raises(ops.KernelError, match="CUDA device"):
        ops.beam_candidates(torch.zeros(4, 18, device=dev), torch.zeros(1, 4), 4)


# ---- the command line -----------------------------------------------------------------------------------------------------

def test_beams_of_the_command_line(beam_cpu_ops, capsys, monkeypatch):
    import sllm_b200.engine.llm as llm_mod
    from sllm_b200.serving import main as cli
    real = llm_mod.LLM
    monkeypatch.setattr(llm_mod, "LLM", lambda model_dir, **kw: real(model_dir, **{**kw, "device": "cpu", "num_pages": 64}))
    common = ["tiny-qwen2", "--mode", "run", "--random-weights", "3", "--prompt-ids", "5,6,7", "--max-new", "4", "--dtype", "float32", "--log-level", "ERROR"]
    assert cli.main(common) == 0
    greedy = capsys.readouterr().out
    assert cli.main(common + ["--beams", "1"]) == 0
    assert capsys.readouterr().out == greedy
    assert cli.main(common + ["--beams", "9", "--length-penalty", "0.5"]) == 0
    assert len(capsys.readouterr().out.strip().split(",")) == 4
    for more, word in ((["--beams", "40"], "beams"), (["--beams", "2", "--temperature", "0.5"], "temperature"), (["--beams", "0"], "beams")):
        with pytest.raises(SystemExit) as e:
            cli.main(common + more)
        assert word in str(e.value)


def test_stop_ids_and_the_length_penalty_of_the_command_line(beam_cpu_ops, capsys, monkeypatch):
    """A continuation that stops at once has one log-probability, one of four tokens four of about the same: by their sums the first is the better, by their means of a high power the second."""
    import sllm_b200.engine.llm as llm_mod
    from sllm_b200.serving import main as cli
    real = llm_mod.LLM
    monkeypatch.setattr(llm_mod, "LLM", lambda model_dir, **kw: real(model_dir, **{**kw, "device": "cpu", "num_pages": 64}))
    common = ["tiny-qwen2", "--mode", "run", "--random-weights", "3", "--prompt-ids", "5,6,7", "--max-new", "4", "--dtype", "float32", "--log-level", "ERROR"]

    def ids(*more):
        assert cli.main(common + list(more)) == 0
        return [int(x) for x in capsys.readouterr().out.strip().split(",") if x]
    greedy = ids()
    assert len(greedy) == 4
    stop = ["--stop-ids", str(greedy[0])]
    assert ids(*stop) == []
    assert ids("--beams", "3", "--length-penalty", "0", *stop) == []
    found = ids("--beams", "3", "--length-penalty", "5", *stop)
    assert len(found) == 4 and greedy[0] not in found
    for bad, word in (("1,x", "token ids"), ("9999999", "vocabulary"), ("-1", "vocabulary")):
        with pytest.raises(SystemExit, match=word):
            cli.main(common + ["--stop-ids=" + bad])
    with pytest.raises(SystemExit, match="float32"):
        cli.main(common + ["--beams", "3", "--length-penalty", "40"])
