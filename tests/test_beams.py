"""Beams on the CPU: requests that share pages, and the search over them, with the kernels replaced by their plain references."""
import itertools
import math
import random

import numpy as np
import pytest
import torch

from garuda_b200 import ConfigError, Engine, SamplingParams, StepEntry
from garuda_b200.csrc.build import load_host_module
from tests.helpers import TINY, folder_weights, model_dir, random_tokens
from tests.plain import branches_plain, llama_plain
from tests.plain.cpu_ops import CpuOps
from tests.test_extensibility import plain as toy_plain, toy_dir, toy_tokens

host = load_host_module()


class BranchCpuOps(CpuOps):
    MOST_COPIES, MOST_BEAMS = 5, 64         # (few copies a call, so that several calls are made)

    def beam_select(self, logits, scores, best, parents, tokens, ws=None):
        items, beams = scores.shape
        for to, x in zip((best, parents, tokens), branches_plain.beam(logits.numpy().reshape(items, beams, -1), scores.numpy(), best.shape[1])):
            to.copy_(torch.from_numpy(np.ascontiguousarray(x)))

    def copy_entries(self, arrays, source, target, dim=0):
        assert source.shape[0] <= self.MOST_COPIES
        for a in arrays:
            index = source.long()
            a.index_copy_(dim, target.long(), a.index_select(dim, index))


def engine(name, **kw):
    return Engine(model_dir(name), dtype="float32", ops=BranchCpuOps(), cuda_graphs=False, **dict(dict(page_size=8, kv_tokens=512, max_concurrent=8), **kw))


# ------------------------------------------------------------------ pages
def test_fork_shares_full_pages_and_copies_the_open_one():
    m = host.CacheManager([host.GroupConfig(16, 0), host.GroupConfig(16, 6)], 4, 4, 64)
    m.acquire(1)
    m.reserve(1, 10)
    m.commit(1, 10)                                    # pages 0 to 2; the window of 6 has passed page 0
    copies = m.fork(1, 2)
    a, b = ([list(m.block_table_row(r, g)[:3]) for g in (0, 1)] for r in (1, 2))
    assert b[0][:2] == a[0][:2] and b[1][:2] == a[1][:2] and a[1][0] == -1
    assert copies == [(0, a[0][2], b[0][2]), (1, a[1][2], b[1][2])] and b[0][2] != a[0][2]
    assert m.length(2) == 10 and m.reserved_length(2) == 10 and m.free_pages(0) == 16 - 4
    m.check_invariants()
    m.release(1)                                        # what both hold stays
    assert m.free_pages(0) == 16 - 3
    m.check_invariants()
    m.reserve(2, 12)
    m.commit(2, 12)
    assert m.fork(2, 3) == []                           # a full last page: nothing to copy
    m.reserve(3, 13)
    m.reserve(2, 13)
    assert m.block_table_row(2, 0)[3] != m.block_table_row(3, 0)[3]
    m.check_invariants()
    m.release(2)
    m.release(3)
    assert m.free_pages(0) == m.free_pages(1) == 16
    m.check_invariants()


def test_fork_refuses_and_leaves_everything():
    m = host.CacheManager([host.GroupConfig(3, 0), host.GroupConfig(2, 0)], 4, 2, 64)
    with pytest.raises(host.CacheError, match="not known"):
        m.fork(1, 2)
    m.acquire(1)
    m.reserve(1, 6)
    m.commit(1, 6)
    with pytest.raises(host.CacheError, match="already"):
        m.fork(1, 1)
    with pytest.raises(host.OutOfPages, match="group 1"):
        m.fork(1, 2)
    assert m.free_pages(0) == 1 and not m.known(2) and m.free_slots == 1
    m.acquire(5)
    with pytest.raises(host.CacheError, match="slot"):
        m.fork(1, 2)
    m.check_invariants()


@pytest.mark.parametrize("seed", range(4))
def test_random_orders_of_forks_and_releases(seed):
    rng = random.Random(seed)
    m = host.CacheManager([host.GroupConfig(40, 0), host.GroupConfig(30, 9), host.GroupConfig(30, 0, 0, 8)], 4, 7, 60)
    live, new = [], itertools.count()
    for _ in range(400):
        what = rng.randrange(4)
        if what == 0 and m.free_slots:
            live.append(next(new))
            m.acquire(live[-1])
        elif what == 1 and live:
            r = rng.choice(live)
            n = min(60, m.length(r) + rng.randrange(1, 12))
            try:
                m.reserve(r, n)
                m.commit(r, n)
            except host.OutOfPages:
                pass
        elif what == 2 and live:
            r, child = rng.choice(live), next(new)
            try:
                copies = m.fork(r, child)
            except host.CacheError:
                assert not m.known(child)
            else:
                live.append(child)
                assert m.length(child) == m.length(r) and all(a != b for _, a, b in copies)
        elif what == 3 and live:
            m.release(live.pop(rng.randrange(len(live))))
        m.check_invariants()
        # a page that will be written (where the next position goes) has one holder
        nexts = [(g, int(m.block_table_row(r, g)[m.length(r) // 4])) for r in live for g in range(3) if m.length(r) % 4]
        assert len(nexts) == len(set(nexts))
    for r in live:
        m.release(r)
    m.check_invariants()
    assert [m.free_pages(g) for g in range(3)] == [40, 30, 30]


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_forked_requests_go_on_by_themselves(name):
    """Three continuations of one request, forked at a position inside a page and again later, against the plain model."""
    e = engine(name)
    toks = random_tokens(name, 30, 7)
    e.step([StepEntry(1, toks[:21], ())])
    with pytest.raises(ValueError, match="forked"):
        e.cache.fork([(1, 2), (2, 3)], e.ops)
    e.cache.fork([(1, k) for k in range(2, 8)], e.ops)
    for k in (4, 5, 6, 7):
        e.runner.end(k)
    tails = {1: toks[21:25], 2: toks[26:30], 3: toks[22:26]}
    for i in range(4):
        got = e.step([StepEntry(r, [t[i]], [0]) for r, t in tails.items()]).numpy().copy()
    e.cache.fork([(3, 9)], e.ops)
    tails[9] = tails[3] + [5]
    got = np.concatenate([got, e.step([StepEntry(9, [5], [0])]).numpy()])
    w = folder_weights(model_dir(name))
    for row, t in zip(got, tails.values()):
        want = llama_plain.forward(TINY[name][0], w, toks[:21] + t)[-1]
        assert np.abs(row - want).max() <= 2e-5 * np.abs(want).max()
    e.cache.manager.check_invariants()
    for r in tails:
        e.runner.end(r)
    assert e.stats()["pages_free"] == e.stats()["pages_total"]


def fork_a_model_with_states(e):
    """Forked requests of the toy architecture, which keeps a running mean beside its pages, against its plain restatement."""
    toks = toy_tokens(14, 3)
    e.step([StepEntry(1, toks, ())])
    e.cache.fork([(1, 2), (1, 3)], e.ops)
    tails = {1: [5, 9], 2: [7, 1], 3: [5, 2]}
    for i in range(2):
        got = e.step([StepEntry(r, [t[i]], [0]) for r, t in tails.items()]).float().cpu().numpy().copy()
    e.runner.end(1)
    e.cache.fork([(3, 4)], e.ops)                       # into the slot that has just been given back
    last = e.step([StepEntry(4, [8], [0]), StepEntry(3, [6], [0])]).float().cpu().numpy()
    for row, t in zip(list(got) + list(last), list(tails.values()) + [[5, 2, 8], [5, 2, 6]]):
        want = toy_plain(toks + t)[-1]
        assert np.abs(row - want).max() <= 2e-5 * np.abs(want).max()


def test_forked_states():
    fork_a_model_with_states(Engine(toy_dir(), dtype="float32", ops=BranchCpuOps(), page_size=8, max_concurrent=4))


def test_fork_takes_everything_back_when_pages_run_out():
    e = engine("A", kv_tokens=32)
    e.step([StepEntry(1, random_tokens("A", 12, 1), ())])
    with pytest.raises(host.OutOfPages):
        e.cache.fork([(1, 2), (1, 3), (1, 4)], e.ops)
    assert e.stats()["pages_free"] == [2] and not e.cache.manager.known(2)
    e.cache.manager.check_invariants()


# ------------------------------------------------------------------ the search
def test_fork_takes_everything_back_when_a_copy_is_refused():
    e = engine("A")
    e.step([StepEntry(1, random_tokens("A", 11, 1), ())])
    free = [e.cache.manager.free_pages(g) for g in range(len(e.cache.groups))]

    def refuse(*args):
        raise RuntimeError("refused")

    e.ops.copy_entries = refuse
    with pytest.raises(RuntimeError, match="refused"):
        e.cache.fork([(1, 2), (1, 3)], e.ops)
    assert not e.cache.manager.known(2) and not e.cache.manager.known(3)
    assert [e.cache.manager.free_pages(g) for g in range(len(e.cache.groups))] == free
    e.cache.manager.check_invariants()


def plain_search(cfg, weights, prompt, beams, max_tokens, penalty, eos, context):
    """The same search with the whole sequence run anew for every beam."""
    live, done = [([], 0.0)], []
    while True:
        rows = []
        for tokens, score in live:
            x = llama_plain.forward(cfg, weights, prompt + tokens)[-1].astype(np.float64)
            lse = x.max() + math.log(np.exp(x - x.max()).sum())
            rows.append(np.float32(score).astype(np.float64) + (x - lse))
        flat = np.concatenate(rows)
        V = len(rows[0])
        order = np.lexsort((np.arange(flat.size), -flat))[:beams * (1 + len(eos))]
        new = []
        for place, at in enumerate(order):
            if len(new) == beams:
                break
            w, t = divmod(int(at), V)
            if t in eos:
                if place < beams:
                    done.append((live[w][0], flat[at], len(live[w][0]) + 1, "eos"))
            else:
                new.append((live[w][0] + [t], flat[at]))
        why = "length" if len(new[0][0]) >= max_tokens else "context_full" if len(prompt) + len(new[0][0]) >= context else ""
        if why:
            done += [(t, s, len(t), why) for t, s in new]
            break
        live = new
        if len(done) >= beams:
            worst = sorted((s / n ** penalty for _, s, n, _ in done), reverse=True)[beams - 1]
            if max(s for _, s in live) / (max_tokens if penalty > 0 else len(live[0][0])) ** penalty <= worst:
                break
    return sorted(done, key=lambda h: -h[1] / h[2] ** penalty)[:beams]


@pytest.mark.parametrize("name, beams, penalty, eos, context", [("A", 3, 1.0, (), 0), ("B", 4, 0.6, "likely", 0), ("C", 1, 1.0, "likely", 0), ("A", 2, -0.5, "likely", 0),
                                                                ("A", 3, 0.0, (), 17)])
def test_search_agrees_with_the_plain_one(name, beams, penalty, eos, context):
    cfg, w = TINY[name][0], folder_weights(model_dir(name))
    prompts = [random_tokens(name, n, 40 + n) for n in (13, 1, 16)]
    if eos == "likely":           # tokens that beams meet
        x = llama_plain.forward(cfg, w, prompts[0])[-1]
        eos = tuple(int(t) for t in np.argsort(-x)[1:3]) if beams < 4 else (int(np.argsort(-x)[2]),)
    e = engine(name, eos_token_id=eos, prefill_chunk=5, **({"context": context} if context else {}))
    got = e.beam_search(prompts, beams=beams, max_tokens=6, length_penalty=penalty)
    for p, hypotheses in zip(prompts, got):
        want = plain_search(cfg, w, p, beams, 6, penalty, set(eos), context or e.max_context)
        assert [h.tokens for h in hypotheses] == [t for t, *_ in want]
        assert [h.finish_reason for h in hypotheses] == [why for *_, why in want]
        assert np.allclose([h.score for h in hypotheses], [s for _, s, *_ in want], rtol=1e-4, atol=1e-4)
    assert e.cache.manager.live_requests == 0 and e.stats()["pages_free"] == e.stats()["pages_total"]
    e.cache.manager.check_invariants()


def test_one_beam_is_greedy():
    e = engine("A", eos_token_id=())
    prompts = [random_tokens("A", n, n) for n in (5, 9)]
    greedy = e.generate(prompts, SamplingParams.greedy(max_tokens=7))
    assert [h[0].tokens for h in e.beam_search(prompts, beams=1, max_tokens=7)] == [r.tokens for r in greedy]


def test_what_the_search_refuses_and_what_it_leaves_behind():
    e = engine("A", max_concurrent=3, kv_tokens=40)
    for kw, match in ((dict(beams=0), "at least one beam"), (dict(max_tokens=0), "one token"), (dict(beams=4), "max_concurrent"), (dict(beams=65), "at most 64")):
        with pytest.raises(ConfigError, match=match):
            e.beam_search([[1, 2]], **dict(dict(beams=2, max_tokens=2), **kw))
    with pytest.raises(ConfigError, match="at least one token"):
        e.beam_search([[]], beams=2)
    with pytest.raises(ConfigError, match="leave room"):
        e.beam_search([[1] * 128], beams=2)
    with pytest.raises(host.CacheError):          # five pages of eight: three beams of seventeen tokens need six
        e.beam_search([random_tokens("A", 15, 3)], beams=3, max_tokens=20)
    assert e.cache.manager.live_requests == 0 and e.stats()["pages_free"] == [5]
    e.cache.manager.check_invariants()
    assert len(e.beam_search([[3, 4]], beams=3, max_tokens=2)[0]) == 3


def small_vocabulary(vocab, seed):
    """A folder of a model with few tokens, and its configuration."""
    import tempfile
    from garuda_b200.weights import write_random_model
    cfg = dict(TINY["A"][0], vocab_size=vocab)
    folder = tempfile.mkdtemp(prefix="garuda_few_tokens_")
    write_random_model(folder, cfg, seed, scale={"q_proj": 8.0, "k_proj": 8.0, "lm_head": 8.0})
    return cfg, folder


@pytest.mark.parametrize("vocab, beams, ends, seed", [(6, 4, 2, 0), (5, 5, 1, 1), (12, 4, 3, 2), (9, 8, 2, 3)])
def test_search_in_a_vocabulary_smaller_than_its_candidates(vocab, beams, ends, seed):
    """A step has every live beam's continuations to choose from, more than the vocabulary has tokens: end tokens of many beams do not crowd the others out."""
    cfg, folder = small_vocabulary(vocab, seed)
    w, prompt = folder_weights(folder), [1, 3, 2, 4]
    x = llama_plain.forward(cfg, w, prompt)[-1]
    eos = tuple(int(t) for t in np.argsort(-x)[:ends])
    e = Engine(folder, dtype="float32", ops=BranchCpuOps(), cuda_graphs=False, page_size=8, kv_tokens=512, max_concurrent=8, eos_token_id=eos)
    got = e.beam_search([prompt], beams=beams, max_tokens=5, length_penalty=1.0)[0]
    want = plain_search(cfg, w, prompt, beams, 5, 1.0, set(eos), e.max_context)
    assert [(h.tokens, h.finish_reason) for h in got] == [(t, why) for t, _, _, why in want]
    assert np.allclose([h.score for h in got], [s for _, s, *_ in want], rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("after, eos", [(0, ()), (2, ()), (2, "likely")])
def test_search_keeps_what_it_has_where_the_model_gives_no_distribution(after, eos):
    """Logits that hold NaN in every beam: the hypotheses so far come back, marked, behind those that have ended; other prompts' are what they were."""
    prompts = [random_tokens("A", 11, 1), random_tokens("A", 7, 2)]
    if eos:
        x = llama_plain.forward(TINY["A"][0], folder_weights(model_dir("A")), prompts[1])[-1]
        eos = (int(np.argmax(x)),)
    want = engine("A", eos_token_id=eos).beam_search(prompts, beams=2, max_tokens=4)
    until = engine("A", eos_token_id=eos).beam_search(prompts[1:], beams=2, max_tokens=after)[0] if after else None
    e = engine("A", eos_token_id=eos)
    run, steps = e.runner.run, []

    def spoilt(entries, **kw):
        logits = run(entries, **kw)
        if entries[0].want:
            steps.append(len(entries))
            if len(steps) == after + 1:
                logits = logits.clone()
                logits[2 if after else 1:, 5] = float("nan")          # the second prompt's beams
        return logits

    e.runner.run = spoilt
    got = e.beam_search(prompts, beams=2, max_tokens=4)
    key = [[(h.tokens, h.finish_reason, h.score) for h in hypotheses] for hypotheses in (got[0], want[0])]
    assert key[0] == key[1]
    ended = [h for h in got[1] if h.finish_reason == "eos"]
    cut = [h for h in got[1] if h.finish_reason == "error"]
    assert got[1] == ended + cut and cut and bool(ended) == bool(eos)
    if after:
        assert [(h.tokens, h.score) for h in cut] == [(h.tokens, h.score) for h in until if h.finish_reason == "length"][:len(cut)]
    else:
        assert [(h.tokens, h.score) for h in cut] == [([], 0.0)]
    assert e.cache.manager.live_requests == 0 and e.stats()["pages_free"] == e.stats()["pages_total"]
