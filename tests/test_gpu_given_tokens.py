"""Captured one-token steps go on with the token, temperature and key they are given, whatever the step before drew: forks of a sequence each take a token
of their own, and so does the sequence they were made of."""

import pytest

import plain_qwen3 as plain
from gpu_helpers import model_case, runner_for
from starter_b200.engine.batch import FED, StepEntry
from starter_b200.sampling import Sampler
from tiny import random_prompt

pytestmark = pytest.mark.gpu


def best(cfg, w, text):
    return int(plain.plain_forward(cfg, w, text)[-1].argmax())


def test_forks_and_their_sequence_go_on_with_tokens_of_their_own(tmp_path_factory):
    folder, cfg, w = model_case(tmp_path_factory, "B")
    runner = runner_for(tmp_path_factory, "B", "float32")
    sampler, vocab = Sampler(runner.device, runner.status), cfg["vocab_size"]
    text = random_prompt(70, vocab, 5)
    first = runner.open_sequence()
    runner.step([StepEntry(first, text[:-1])])
    drawn = runner.step_and_select([StepEntry(first, [text[-1]], [0])], sampler, [0.0], [0], [0])[0]
    assert drawn == best(cfg, w, text)
    slots = [first] + runner.fork(first, 2)
    others = [(drawn + 1 + i) % vocab for i in range(3)]
    # the sequence itself first: the device still holds what it drew for it
    for slot, token in zip(slots, others):
        assert runner.step_and_select([StepEntry(slot, [token], [0])], sampler, [0.0], [0], [0]) == [best(cfg, w, text + [token])]
    both = runner.step_and_select([StepEntry(s, [7], [0]) for s in slots], sampler, [0.0] * 3, [0] * 3, [0] * 3)
    assert both == [best(cfg, w, text + [token, 7]) for token in others]
    for s in slots:
        runner.close_sequence(s)
    runner.check_status()


def test_a_token_that_was_not_drawn(tmp_path_factory):
    folder, cfg, w = model_case(tmp_path_factory, "A")
    runner = runner_for(tmp_path_factory, "A", "float32")
    sampler, vocab = Sampler(runner.device, runner.status), cfg["vocab_size"]
    text, slot = random_prompt(20, vocab, 6), runner.open_sequence()
    runner.step([StepEntry(slot, text)])
    given = 11
    for turn in range(8):
        text = text + [given]
        handle = runner.start_step([StepEntry(slot, [given], [0])], sampler, [0.0], [0], [0])
        want = best(cfg, w, text)
        if turn == 5:
            given = (want + 3) % vocab                   # the drawn token has not been read
        else:
            got = handle.result()
            assert got == [want]
            got[0] = want if turn % 2 else (want + 5) % vocab            # (in the list that was handed out)
            given = got[0]
    handle = runner.start_step([StepEntry(slot, [given], [0])], sampler, [0.0], [0], [0])
    text = text + [given]
    ahead = runner.start_step([StepEntry(slot, [FED], [0])], sampler, [0.0], [0], [0])
    got = handle.result()
    assert got == [best(cfg, w, text)]
    text = text + got
    assert ahead.result() == [best(cfg, w, text)]
    runner.close_sequence(slot)
    runner.check_status()


def test_settings_that_change_between_steps(tmp_path_factory):
    """The same tokens at another temperature or key: what a runner without captured steps draws."""
    from starter_b200.engine import ModelRunner, load_model

    folder, cfg, w = model_case(tmp_path_factory, "A")
    model = load_model(folder, "float32")
    drawn = []
    for graphs in (True, False):
        runner = ModelRunner(model, max_tokens=64 * 4, max_sequences=2, use_graphs=graphs)
        sampler, slot, out = Sampler(runner.device, runner.status), runner.open_sequence(), []
        token = 5
        for turn, (temperature, key) in enumerate([(0.0, 0), (0.9, 3), (0.9, 3), (2.0, 3), (2.0, 8), (0.0, 8), (1.5, 9)]):
            token = int(runner.step_and_select([StepEntry(slot, [token], [0])], sampler, [temperature], [key], [turn + 1])[0])
            out.append(token)
        drawn.append(out)
    assert drawn[0] == drawn[1]


def test_settings_that_change_where_the_device_holds_the_tokens(tmp_path_factory):
    """Steps that go on from the device (FED) at another temperature or key, against steps that are given what was drawn."""
    runner = runner_for(tmp_path_factory, "A", "float32")
    sampler, drawn = Sampler(runner.device, runner.status), []
    for fed in (True, False):
        slot, token, out = runner.open_sequence(), 5, []
        for turn, (temperature, key) in enumerate([(0.0, 0), (0.9, 3), (0.9, 3), (2.0, 3), (2.0, 8), (0.0, 8), (1.5, 9)]):
            token = int(runner.step_and_select([StepEntry(slot, [FED if fed and turn else token], [0])], sampler, [temperature], [key], [turn + 1])[0])
            out.append(token)
        drawn.append(out)
        runner.close_sequence(slot)
    assert drawn[0] == drawn[1]


def test_some_tokens_given_and_some_held(tmp_path_factory):
    folder, cfg, w = model_case(tmp_path_factory, "A")
    runner = runner_for(tmp_path_factory, "A", "float32")
    sampler, vocab = Sampler(runner.device, runner.status), cfg["vocab_size"]
    texts = [random_prompt(n, vocab, n) for n in (9, 33)]
    slots = [runner.open_sequence() for _ in texts]
    runner.step([StepEntry(s, t[:-1]) for s, t in zip(slots, texts)])
    args = sampler, [0.0] * 2, [0] * 2, [0] * 2
    first = runner.start_step([StepEntry(s, [t[-1]], [0]) for s, t in zip(slots, texts)], *args)
    want = [best(cfg, w, t) for t in texts]
    held = list(runner.cache.lengths)
    with pytest.raises(ValueError, match="device-held"):
        runner.start_step([StepEntry(slots[0], [FED], [0]), StepEntry(slots[1], [(want[1] + 1) % vocab], [0])], *args)
    assert runner.cache.lengths == held and first.result() == want
    first.result()[1] = -5                               # (the list is the caller's to change)
    # the drawn one given back is the one that is held
    second = runner.start_step([StepEntry(slots[0], [FED], [0]), StepEntry(slots[1], [want[1]], [0])], *args)
    assert second.result() == [best(cfg, w, t + [x]) for t, x in zip(texts, want)]
    for s in slots:
        runner.close_sequence(s)
    runner.check_status()
