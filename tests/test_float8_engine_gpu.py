"""Serving in 8 bits through the engine: generation, graphs, portions, the command line's replay, against the plain model."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from tests.helpers import ROOT, TINY, folder_weights, model_dir, plain_logits, random_tokens
from tests.plain import float8_plain, llama_plain

pytestmark = pytest.mark.gpu


def engine(name, **kw):
    from garuda_b200 import Engine
    args = dict(dtype="bfloat16", page_size=32, max_concurrent=4, max_batch_tokens=64, prefill_chunk=40)
    args.update(kw)
    return Engine(model_dir(name, torch.bfloat16), **args)


def logits_of(e, tokens, portions):
    """Logits of every position of one request that goes in by these portions."""
    from garuda_b200.engine.step import StepEntry
    rows, at = [], 0
    for n in portions:
        part = tokens[at:at + n]
        rows.append(e.runner.run([StepEntry(7, part, list(range(len(part))))]).float().cpu())
        at += n
    e.cache.release(7)
    return torch.cat(rows).numpy()


def quantised(weights, config):
    """The folder's weights with the layers' matrices rounded to 8 bits as they are held (stacked as the engine stacks them)."""
    out = dict(weights)
    for l in range(config["num_hidden_layers"]):
        p = f"model.layers.{l}."
        for group in (("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj"), ("self_attn.o_proj",), ("mlp.gate_proj", "mlp.up_proj"),
                      ("mlp.down_proj",)):
            mats = [torch.from_numpy(weights[p + n + ".weight"]) for n in group]
            codes, scales = float8_plain.weight(torch.cat(mats))
            N, K = codes.shape
            w = (codes * scales.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]).float()
            for n, part in zip(group, w.split([m.shape[0] for m in mats])):
                out[p + n + ".weight"] = part.numpy()
    return out


def off(got, want):
    return float(np.linalg.norm(got - want) / np.linalg.norm(want))


# An E4M3 number is off by 2^-4 of itself at most, by 2^-5.6 in the mean square (a uniform error in a step of 2^-3 of the power of two below). A
# layer adds a few such errors (values, the projections' tokens) to a residual that they are a part of: 2^-4 of the logits for the
# cache, twice that with tokens in 8 bits is above what two or three layers can gather, and far below a wrong page, scale or row.
CACHE_OFF, BOTH_OFF = 2.0 ** -4, 2.0 ** -3


@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E"])
def test_logits(name):
    tokens = random_tokens(name, 90, 5)
    cfg = TINY[name][0]
    w = folder_weights(model_dir(name, torch.bfloat16))
    want = plain_logits(name, torch.bfloat16, tokens)
    cache = engine(name, cache_dtype="float8_e4m3")
    got = logits_of(cache, tokens, [90])
    assert off(got, want) <= CACHE_OFF
    single = logits_of(cache, tokens, [37, 3] + [1] * 50)          # the same in portions and single tokens, from graphs
    assert off(single, want) <= CACHE_OFF
    assert cache.runner.graphs.replays > 0
    both = engine(name, cache_dtype="float8_e4m3", weight_dtype="float8_e4m3")
    held = llama_plain.forward(cfg, quantised(w, cfg), tokens)
    assert off(logits_of(both, tokens, [60, 30]), held) <= BOTH_OFF
    weights = engine(name, weight_dtype="float8_e4m3")
    assert off(logits_of(weights, tokens, [33] + [1] * 57), held) <= BOTH_OFF
    for e in (cache, both, weights):
        e.check_errors()


def test_32_bit_model_over_a_cache_in_8_bits():
    tokens = random_tokens("D", 80, 6)
    from garuda_b200 import Engine
    e = Engine(model_dir("D"), dtype="float32", page_size=32, cache_dtype="float8_e4m3")
    assert off(logits_of(e, tokens, [50, 1, 1, 28]), plain_logits("D", torch.float32, tokens)) <= CACHE_OFF


@pytest.mark.parametrize("name", ["D", "E"])
def test_generation_from_graphs_is_generation_without(name):
    from garuda_b200 import SamplingParams
    prompts = [random_tokens(name, n, 60 + n) for n in (9, 64, 1, 130, 33)]
    results = []
    for graphs in (True, False):
        e = engine(name, cache_dtype="float8_e4m3", weight_dtype="float8_e4m3", cuda_graphs=graphs, prefill_chunk=0, max_batch_tokens=512)
        results.append([r.tokens for r in e.generate(prompts, SamplingParams.greedy(max_tokens=40))])
        st = e.stats()
        assert st["completed"] == len(prompts) and st["pages_free"] == st["pages_total"]
        e.check_errors()
    assert results[0] == results[1] and all(len(t) == 40 for t in results[0])


def test_an_8_bit_cache_holds_twice_the_positions():
    from garuda_b200 import Engine
    args = dict(dtype="bfloat16", kv_cache_bytes=1 << 20)
    plain, small = Engine(model_dir("E", torch.bfloat16), **args), Engine(model_dir("E", torch.bfloat16), cache_dtype="float8_e4m3", **args)
    assert small.stats()["pages_total"][0] >= 1.9 * plain.stats()["pages_total"][0]


def test_replay_from_the_command_line(tmp_path):
    tokens = random_tokens("D", 40, 8)
    steps = [{"step": 0, "entries": [{"id": "a", "tokens": tokens[:33], "want": [32]}], "end": []},
             {"step": 1, "entries": [{"id": "a", "tokens": tokens[33:34], "want": [0]}], "end": ["a"]}]
    cmd = [sys.executable, os.path.join(ROOT, "bin", "trace_run"), "--model", model_dir("D", torch.bfloat16), "--dtype", "bfloat16", "--out",
           str(tmp_path), "--max-tokens", "256", "--cache-dtype", "float8_e4m3", "--weight-dtype", "float8_e4m3"]
    done = subprocess.run(cmd, input="\n".join(json.dumps(s) for s in steps) + "\n", text=True, capture_output=True, timeout=600)
    assert done.returncode == 0, done.stderr
    cfg = TINY["D"][0]
    held = llama_plain.forward(cfg, quantised(folder_weights(model_dir("D", torch.bfloat16)), cfg), tokens[:34])
    for step, row in ((0, 32), (1, 33)):
        got = np.fromfile(next(str(p) for p in tmp_path.iterdir() if p.name.startswith(f"{step}.")), dtype=np.float32)
        assert off(got, held[row]) <= BOTH_OFF


@pytest.mark.parametrize("graphs", [True, False])
def test_preemption_over_a_cache_in_8_bits(graphs):
    """A pool too small for all requests: some are sent back and start again, in pages that others have used. What pages held and what scales they
    had counts for nothing (codes that are no numbers and scales of 2^60 to begin with). A request that starts again goes in at once with
    what it had got token by token, whose codes may differ; so every chosen token is held against the plain model: its logit is the
    largest but for what the cache's codes move two logits by."""
    from garuda_b200 import Engine, SamplingParams
    prompts = [random_tokens("A", 20, 70 + i) for i in range(3)]
    tight = Engine(model_dir("A", torch.bfloat16), dtype="bfloat16", page_size=8, kv_tokens=96, max_concurrent=3, cuda_graphs=graphs,
                   cache_dtype="float8_e4m3")
    for pool, scales in zip(tight.cache.k_pools + tight.cache.v_pools, tight.cache.k_scales + tight.cache.v_scales):
        pool.view(torch.uint8).fill_(0x7F)
        scales.fill_(2.0 ** 60)
    got = tight.generate(prompts, SamplingParams.greedy(max_tokens=24))
    st = tight.stats()
    assert st["preemptions"] > 0 and st["completed"] == len(prompts) and st["pages_free"] == st["pages_total"]
    cfg = TINY["A"][0]
    w = folder_weights(model_dir("A", torch.bfloat16))
    for prompt, r in zip(prompts, got):
        assert len(r.tokens) == 24
        want = llama_plain.forward(cfg, w, prompt + r.tokens[:-1])
        assert off(logits_of(tight, prompt + r.tokens[:-1], [20, 20] + [1] * 3), want) <= CACHE_OFF        # in the same pages, once more
        rows = want[len(prompt) - 1:]
        assert (rows.max(1) - rows[np.arange(24), r.tokens] <= 2 * CACHE_OFF * np.linalg.norm(rows, axis=1)).all()
    tight.check_errors()
