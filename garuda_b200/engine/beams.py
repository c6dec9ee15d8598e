"""Beam search through the step function: every beam is a request of its own over shared pages.

A step runs one token of every live beam, as a decode step does; ``beam_select`` chooses among all continuations of an item's beams; a
beam that goes on in several ways is forked (``PagedCache.fork``), one that goes on in none is released. The reference samples one
continuation per request (garuda/src/runtime/mod.rs:698-760); this is beside it.
"""
from __future__ import annotations

import itertools
from dataclasses import dataclass, field
from typing import List, Sequence

import torch

from ..config.model_config import ConfigError
from .step import StepEntry

_REQUESTS = itertools.count(1 << 40)        # ids that no scheduler hands out


@dataclass
class Hypothesis:
    """A continuation of a prompt: its tokens (without the token that ended it), the sum of their log-probabilities (with that token's), and why it
    ended: "eos", "length" or "context_full"; or "error": the model gave none of its beams a distribution (logits with an infinity or NaN), and these are
    the tokens in front of that."""
    tokens: List[int] = field(default_factory=list)
    score: float = 0.0
    finish_reason: str = ""


class _Item:
    """One prompt's search."""

    def __init__(self, prompt, beams):
        self.prompt, self.beams = prompt, beams
        self.live, self.done = [], []               # hypotheses
        self.requests, self.next = [], []           # of the live ones: their requests and the tokens that these run next

    def penalised(self, h: Hypothesis, length_penalty: float) -> float:
        return h.score / (len(h.tokens) + (h.finish_reason == "eos")) ** length_penalty


def beam_search(engine, prompts: Sequence[Sequence[int]], beams: int, max_tokens: int, length_penalty: float) -> List[List[Hypothesis]]:
    ops, cache = engine.ops, engine.cache
    vocab = engine.model.spec.vocab_size
    # as many candidates as leave enough that do not end the text, whichever do (a step may have fewer)
    candidates = beams * (1 + len(engine.eos_ids))
    most = getattr(ops, "MOST_BEAMS", 64)
    if beams < 1 or max_tokens < 1:
        raise ConfigError(f"beam search needs at least one beam and one token, not {beams} and {max_tokens}")
    if candidates > most or beams > vocab:
        raise ConfigError(f"{beams} beams of a model with {len(engine.eos_ids)} end tokens need {candidates} candidates "
                          f"(at most {most}, and no more beams than the vocabulary's {vocab} tokens)")
    if beams > cache.config.max_requests:
        raise ConfigError(f"{beams} beams need as many slots, the engine has {cache.config.max_requests} (max_concurrent)")
    for p in prompts:
        if not len(p):
            raise ConfigError("a prompt must hold at least one token")
        if len(p) >= engine.max_context:
            raise ConfigError(f"a prompt of {len(p)} tokens does not leave room in a context of {engine.max_context}")
    out = [None] * len(prompts)
    waiting = [(i, _Item([int(t) for t in p], beams)) for i, p in enumerate(prompts)]
    running = []
    try:
        while waiting or running:
            # as many items as there are slots for all their beams
            while waiting and (len(running) + 1) * beams <= cache.config.max_requests:
                i, item = waiting.pop(0)
                running.append((i, item))
                _begin(engine, item)
            _step(engine, [item for _, item in running], candidates, max_tokens, length_penalty)
            for i, item in running:
                if not item.live:
                    # (stable: equal ones as they ended; those that have not ended come last, one behind the other by their scores)
                    order = sorted(item.done, key=lambda h: (1, -h.score) if h.finish_reason == "error" else (0, -item.penalised(h, length_penalty)))
                    out[i] = order[:beams]
            running = [(i, item) for i, item in running if item.live]
    finally:
        for _, item in running:
            _end(engine, item.requests)
    return out


def _end(engine, requests) -> None:
    for r in requests:
        if engine.cache.manager.known(r):          # (a request is, once a step has run a token of it)
            engine.runner.end(r)


def _begin(engine, item) -> None:
    """The prompt runs in portions, but for its last token, which is the first beam's next one."""
    request = next(_REQUESTS)
    item.requests, item.live = [request], [Hypothesis()]
    item.next = [item.prompt[-1]]
    front, portion = item.prompt[:-1], engine.prefill_chunk
    for i in range(0, len(front), portion):
        engine.runner.run([StepEntry(request, front[i:i + portion], ())])


def _step(engine, items, candidates, max_tokens, length_penalty) -> None:
    ops = engine.ops
    entries = [StepEntry(r, (t,), (0,)) for item in items for r, t in zip(item.requests, item.next)]
    logits = engine.runner.run(entries)
    # items in their first step have one beam: one call for them, one for the others
    at, chosen = 0, {}
    rows = []
    for item in items:
        rows.append(range(at, at + len(item.live)))
        at += len(item.live)
    for count in sorted({len(item.live) for item in items}):
        group = [k for k, item in enumerate(items) if len(item.live) == count]
        n = min(candidates, count * engine.model.spec.vocab_size)
        index = [r for k in group for r in rows[k]]
        part = logits if len(index) == at else logits[torch.tensor(index, device=logits.device)]
        scores = torch.tensor([[h.score for h in items[k].live] for k in group], dtype=torch.float32).to(logits.device)
        best = torch.empty(len(group), n, dtype=torch.float32, device=logits.device)
        parents, tokens = (torch.empty(len(group), n, dtype=torch.int32, device=logits.device) for _ in range(2))
        ops.beam_select(part, scores, best, parents, tokens)
        for k, b, p, t in zip(group, best.tolist(), parents.tolist(), tokens.tolist()):
            chosen[k] = list(zip(b, p, t))
    engine.check_errors()
    for k, item in enumerate(items):
        _choose(engine, item, chosen[k], max_tokens, length_penalty)


def _choose(engine, item, candidates, max_tokens, length_penalty) -> None:
    """The item's beams of the next step, from its best continuations in order."""
    cache, beams = engine.cache, item.beams
    live, parents = [], []
    full = cache.manager.length(item.requests[0]) + 1 >= engine.max_context          # with the token that is chosen now
    for place, (score, parent, token) in enumerate(candidates):
        if score == float("-inf") or len(live) == beams:
            break
        before = item.live[parent]
        if token in engine.eos_ids:
            # (one that is not among the best now would not be among them as a hypothesis)
            if place < beams:
                item.done.append(Hypothesis(list(before.tokens), score, "eos"))
            continue
        h = Hypothesis(before.tokens + [token], score)
        h.finish_reason = "length" if len(h.tokens) >= max_tokens else "context_full" if full else ""
        live.append(h)
        parents.append(parent)
    ended = [h for h in live if h.finish_reason]           # (all of them or none: beams are of one length)
    if candidates[0][0] == float("-inf"):
        item.done += [Hypothesis(h.tokens, h.score, "error") for h in item.live]
    if ended or not live:
        item.done += ended
        live = []
    elif len(item.done) >= beams:
        # enough have ended, and no beam can overtake the worst of the best any more: its score only falls (and is divided by more at most once
        # its length is the largest)
        worst = sorted((item.penalised(h, length_penalty) for h in item.done), reverse=True)[beams - 1]
        length = max_tokens if length_penalty > 0 else len(live[0].tokens)
        if max(h.score for h in live) / length ** length_penalty <= worst:
            live = []
    requests = item.requests
    if not live:
        _end(engine, requests)
        item.requests, item.live = [], []
        return
    # a beam's first continuation takes its request over; those that have none are released, whose slots and pages the others' copies may need
    kept, heirs, forks = {}, [], []
    for parent in parents:
        if parent not in kept:
            kept[parent] = requests[parent]
            heirs.append(requests[parent])
        else:
            child = next(_REQUESTS)
            heirs.append(child)
            forks.append((requests[parent], child))
    _end(engine, [r for w, r in enumerate(requests) if w not in kept])
    item.requests = list(kept.values())
    cache.fork(forks, engine.ops)
    item.requests, item.live, item.next = heirs, live, [h.tokens[-1] for h in live]
