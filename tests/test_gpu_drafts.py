"""Steps with drafted trees, forks and scores together, on whole models: what they give is what one-token steps and the plain
implementation give."""

import numpy as np
import pytest
import torch

import plain_qwen3 as plain
from gpu_helpers import BF16_TOL, DTYPES, FP32_TOL, model_case, runner_for
from starter_b200.engine.batch import StepEntry, TreeEntry
from starter_b200.sampling import Sampler, SamplingParams
from starter_b200.sampling.sampler import request_key
from tiny import random_prompt

pytestmark = pytest.mark.gpu


def draft(rng, root, truth, vocab, nodes):
    """A tree behind ``root``: the first tokens of ``truth`` as a chain through it, wrong tokens around."""
    tokens, parents, tip = [root], [-1], 0
    right = int(rng.integers(0, min(len(truth), nodes - 1) + 1)) if nodes > 1 else 0
    while len(tokens) < nodes:
        if right and rng.random() < 0.6:
            depth, at = 0, tip
            while at > 0:
                depth, at = depth + 1, parents[at]
            tokens.append(truth[depth])
            parents.append(tip)
            tip = len(tokens) - 1
            right -= 1
        else:
            tokens.append(int(rng.integers(0, vocab)))
            parents.append(int(rng.integers(0, len(tokens) - 1)))
    return tokens, parents


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_drafted_steps_draw_what_single_tokens_draw(tmp_path_factory, name):
    """Greedy, float32: three unequal sequences, trees of 1 to 40 nodes, against the plain implementation's continuation."""
    folder, cfg, w = model_case(tmp_path_factory, name)
    runner = runner_for(tmp_path_factory, name, "float32")
    vocab, rng = cfg["vocab_size"], np.random.default_rng(3)
    prompts = [random_prompt(n, vocab, 70 + n) for n in (5, 60, 130)]
    new = 40
    want = [plain.plain_generate(cfg, w, p, new + 8) for p in prompts]
    sampler = Sampler(runner.device, runner.status)
    slots = [runner.open_sequence() for _ in prompts]
    try:
        logits = runner.step([StepEntry(s, p, [len(p) - 1]) for s, p in zip(slots, prompts)])
        out = [[t] for t in sampler.select(logits, [0.0] * 3, [0] * 3, [0] * 3)]
        steps = kept = 0
        while min(len(o) for o in out) < new:
            live = [i for i in range(3) if len(out[i]) < new]
            entries = []
            for i in live:
                n = int(rng.choice([1, 2, 9, 17, 40]))
                entries.append(TreeEntry(slots[i], *draft(rng, out[i][-1], want[i][len(out[i]):], vocab, n)))
            for i, got in zip(live, runner.step_trees(entries, sampler, [0.0] * len(live), [0] * len(live))):
                assert len(got) >= 1
                out[i] += got
                kept += len(got)
                assert runner.cache.lengths[slots[i]] == len(prompts[i]) + len(out[i]) - 1
            steps += len(live)
        runner.check_status()
        assert kept > steps                     # drafts were accepted
        for o, wanted in zip(out, want):
            assert o[:new] == wanted[:new]
        # what the cache holds now is what the tokens say: the next logits are the plain implementation's
        logits = runner.step([StepEntry(s, [o[-1]], [0]) for s, o in zip(slots, out)])
        for row, prompt, o in zip(logits, prompts, out):
            full = plain.plain_forward(cfg, w, prompt + o)[-1]
            assert (row.cpu() - full).abs().max() <= FP32_TOL * full.abs().max()
        runner.cache.check()
    finally:
        for s in slots:
            runner.close_sequence(s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_node_has_the_logits_of_its_way(tmp_path_factory, dtype):
    """A tree's logits, node by node, against the plain implementation on the tokens of its way."""
    folder, cfg, w = model_case(tmp_path_factory, "B")
    runner = runner_for(tmp_path_factory, "B", dtype)
    vocab, rng = cfg["vocab_size"], np.random.default_rng(4)
    prompts = [random_prompt(n, vocab, 80 + n) for n in (61, 7)]
    slots = [runner.open_sequence() for _ in prompts]
    try:
        runner.step([StepEntry(s, p) for s, p in zip(slots, prompts)])
        entries = [TreeEntry(s, *draft(rng, 3, random_prompt(9, vocab, 1), vocab, n)) for s, n in zip(slots, (30, 5))]
        ctx = runner.make_context(entries, trees=True)
        logits = runner.model.forward(ctx, ctx.want_rows).cpu()
        row = 0
        for prompt, e in zip(prompts, entries):
            for i in range(len(e.tokens)):
                way, at = [], i
                while at >= 0:
                    way.append(e.tokens[at])
                    at = e.parents[at]
                full = plain.plain_forward(cfg, w, prompt + way[::-1])[-1]
                assert (logits[row] - full).abs().max() <= (FP32_TOL if dtype == "float32" else BF16_TOL) * full.abs().max()
                row += 1
    finally:
        for s in slots:
            runner.close_sequence(s)


def test_drafted_steps_at_a_temperature(tmp_path_factory):
    """The draw behind a node is a function of the request's key and the position: with drafts or without, the same tokens."""
    from starter_b200 import Engine

    folder, cfg, _ = model_case(tmp_path_factory, "A")
    vocab, prompt, new = cfg["vocab_size"], random_prompt(20, cfg["vocab_size"], 5), 30
    engine = Engine(folder, dtype="float32", max_batch=2, max_tokens=64 * 12)
    want = engine.complete([prompt], new, temperature=0.9, seed=11)[0].tokens
    runner, sampler, rng = engine.runner, engine.sampler, np.random.default_rng(6)
    key = request_key(SamplingParams(0.9, 11).seed, 0)
    slot = runner.open_sequence()
    logits = runner.step([StepEntry(slot, prompt, [len(prompt) - 1])])
    out = sampler.select(logits, [0.9], [key], [len(prompt)])
    while len(out) < new:
        tokens, parents = draft(rng, out[-1], want[len(out):] or [0], vocab, int(rng.integers(1, 20)))
        out += runner.step_trees([TreeEntry(slot, tokens, parents)], sampler, [0.9], [key])[0]
    assert out[:new] == want
    runner.close_sequence(slot)
    engine.runner.cache.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_forks_go_on_by_themselves(tmp_path_factory, dtype):
    """A prompt run once, forked, each fork continued with tokens of its own (drafts too): as if each had run alone."""
    folder, cfg, w = model_case(tmp_path_factory, "B")
    runner = runner_for(tmp_path_factory, "B", dtype)
    vocab, tol = cfg["vocab_size"], FP32_TOL if dtype == "float32" else BF16_TOL
    sampler = Sampler(runner.device, runner.status)
    for length in (64, 100):
        prompt = random_prompt(length, vocab, length)
        first = runner.open_sequence()
        runner.step([StepEntry(first, prompt)])
        slots = [first] + runner.fork(first, 3)
        texts = [prompt + random_prompt(3 + 40 * i, vocab, 90 + i) for i in range(4)]
        logits = runner.step([StepEntry(s, t[length:], [len(t) - length - 1]) for s, t in zip(slots, texts)])
        runner.close_sequence(first)                       # its pages stay with those that share them
        slots, texts, rows = slots[1:], texts[1:], logits[1:].cpu()
        for row, t in zip(rows, texts):
            full = plain.plain_forward(cfg, w, t)[-1]
            assert (row - full).abs().max() <= tol * full.abs().max()
        got = runner.step_trees([TreeEntry(s, [1, 2, 3], [-1, 0, 0]) for s in slots], sampler, [0.0] * 3, [0] * 3)
        after = runner.step([StepEntry(s, [g[-1]], [0]) for s, g in zip(slots, got)]).cpu()
        for row, t, g in zip(after, texts, got):
            full = plain.plain_forward(cfg, w, t + [1] + g)[-1]
            assert (row - full).abs().max() <= tol * full.abs().max()
        part = runner.fork(slots[0], 1, length=70 if length == 100 else 64)[0]
        held = runner.cache.lengths[part]
        row = runner.step([StepEntry(part, [9], [0])])[0].cpu()
        full = plain.plain_forward(cfg, w, texts[0][:held] + [9])[-1]
        assert (row - full).abs().max() <= tol * full.abs().max()
        runner.cache.check()
        for s in slots + [part]:
            runner.close_sequence(s)
        runner.cache.check()
    runner.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["A", "C"])
def test_scores_of_texts(tmp_path_factory, name, dtype):
    """Log probabilities, entropies and alternatives of unequal texts through ``Engine.score``."""
    from starter_b200 import Engine

    folder, cfg, w = model_case(tmp_path_factory, name)
    engine = Engine(folder, dtype=dtype, max_batch=3)
    texts = [random_prompt(n, cfg["vocab_size"], 100 + n) for n in (1, 2, 65, 200, 9)]
    tol = FP32_TOL if dtype == "float32" else BF16_TOL
    for top in (0, 4):
        got = engine.score(texts, top=top)
        assert len(got) == len(texts)
        for s, text in zip(got, texts):
            assert len(s.logprobs) == len(s.entropies) == len(s.top_ids) == len(s.top_logprobs) == len(text) - 1
            logits = plain.plain_forward(cfg, w, text)[:-1].double()
            if len(text) == 1:
                continue
            off = 2 * tol * logits.abs().max()             # both the logit and the sum of exponentials are off by a logit's error
            logp = torch.log_softmax(logits, 1)
            want = logp.gather(1, torch.tensor(text[1:])[:, None])[:, 0]
            assert (torch.tensor(s.logprobs) - want).abs().max() <= off
            assert (torch.tensor(s.entropies) + (logp.exp() * logp).sum(1)).abs().max() <= 4 * off
            for ids, values, row in zip(s.top_ids, s.top_logprobs, logp):
                assert len(ids) == len(values) == top and len(set(ids)) == top
                if top:
                    best = torch.topk(row, top).values
                    assert (torch.tensor(values) - best).abs().max() <= off and (row[ids] - best).abs().max() <= 2 * off
    assert engine.score([]) == []
    engine.runner.cache.check()
    assert engine.runner.cache.slots.held_count == 0


def test_what_cannot_be_drafted_or_scored(tmp_path_factory):
    from starter_b200 import Engine
    from tiny_kesedra import make_kesedra_folder

    runner = runner_for(tmp_path_factory, "A", "float32")
    sampler = Sampler(runner.device, runner.status)
    slot = runner.open_sequence()
    runner.step([StepEntry(slot, [1, 2, 3])])
    for entry in (TreeEntry(slot, [1, 2], [-1]), TreeEntry(slot, [1, 2], [-1, 1]), TreeEntry(slot, [1, 999999], [-1, 0]), TreeEntry(slot, [], [])):
        with pytest.raises(ValueError):
            runner.step_trees([entry], sampler, [0.0], [0])
        assert runner.cache.lengths[slot] == 3
    with pytest.raises(ValueError):
        runner.step_trees([TreeEntry(slot, [1], [-1])], sampler, [0.0, 0.0], [0])
    with pytest.raises(ValueError):
        runner.score([[]])
    with pytest.raises(ValueError):
        runner.score([[1, 2]], top=33)
    runner.close_sequence(slot)
    runner.cache.check()
    folder = make_kesedra_folder(tmp_path_factory.mktemp("recurrent"), "KA")
    engine = Engine(folder, dtype="float32", max_tokens=256)
    slot = engine.runner.open_sequence()
    with pytest.raises(ValueError, match="cannot see"):
        engine.runner.step_trees([TreeEntry(slot, [1], [-1])], sampler, [0.0], [0])
    # a fork of a model with states goes on as the sequence itself does
    engine.runner.step([StepEntry(slot, [1, 2, 3, 4])])
    new = engine.runner.fork(slot)[0]
    a, b = engine.runner.step([StepEntry(slot, [7, 8], [1]), StepEntry(new, [7, 8], [1])])
    assert torch.equal(a, b)
    assert engine.score([[1, 2, 3]])[0].logprobs
