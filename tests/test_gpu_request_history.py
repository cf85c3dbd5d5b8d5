"""What the penalties' histories hold on the device, whichever steps took a sequence's tokens, and whether steps on a guess
are used where rows have rules."""
import numpy as np
import pytest
import torch

import plain_requests as plain
import tiny

pytestmark = pytest.mark.gpu


@pytest.fixture
def engine(tiny_folders):
    from foundry_b200 import Engine
    return Engine.from_folder(tiny_folders["tiny_b"], dtype="float32", max_tokens=2048, max_slots=4)


def params(**more):
    from foundry_b200 import SamplingParams
    return SamplingParams(0.8, 3, **more)


def step(slot, tokens):
    from foundry_b200 import SequenceStep
    return SequenceStep(slot, list(tokens), [len(tokens) - 1])


def assert_holds(engine, slot, prompt, said):
    V = engine.spec.vocab_size
    engine._settle()
    want = plain.counts_of(prompt, said, V)
    history = engine.token_history()
    assert np.array_equal(history.counts[slot].cpu().numpy(), want)
    assert np.array_equal(history.seen[slot].cpu().numpy(), plain.pack_bits(want[None] != 0)[0])


@pytest.mark.parametrize("pieces", [[9, 30, 4], [1, 1, 20], [70, 1]])
def test_pieces_of_a_prompt(engine, pieces):
    from foundry_b200 import SequenceStep
    V, p = engine.spec.vocab_size, params(repetition_penalty=1.4)
    for sequence in range(2):
        prompt = tiny.random_tokens(60 + sequence, sum(pieces), V)
        slot, at = engine.open_sequence(), 0
        for n in pieces[:-1]:
            engine.step([SequenceStep(slot, prompt[at:at + n], [n - 1] if n == 1 else [])])
            at += n
        tokens = engine.step_select([step(slot, prompt[at:])], p, [0], [0])
        assert_holds(engine, slot, prompt, [])
        said = []
        for count in range(1, 6):
            said += tokens
            tokens = engine.step_select([step(slot, tokens)], p, [0], [count], count < 5)
        assert_holds(engine, slot, prompt, said)
        engine.close_sequence(slot)


def test_a_penalty_that_comes_later(engine):
    V, prompt = engine.spec.vocab_size, [5, 5, 9]
    slot, other = engine.open_sequence(), engine.open_sequence()
    tokens = engine.step_select([step(slot, prompt), step(other, [4])], params(), [0, 1], [0, 0], True)
    said = [[], []]
    for count, rules in enumerate([params(), params(), params(top_k=5), params(presence_penalty=0.5), params(), params(),
                                   params(presence_penalty=0.5)], 1):
        for mine, t in zip(said, tokens):
            mine.append(t)
        tokens = engine.step_select([step(slot, tokens[:1]), step(other, tokens[1:])], [rules, params(top_p=0.9)], [0, 1],
                                    [count] * 2, True)
    assert_holds(engine, slot, prompt, said[0])
    assert engine.tokens_said(slot) == said[0] and engine.tokens_said(other) == said[1]
    assert max(said[0]) < V


def test_a_session_behind_steps_of_a_prompt(engine):
    prompt = tiny.random_tokens(3, 40, engine.spec.vocab_size)
    slot = engine.open_sequence()
    engine.step([step(slot, prompt[:25])])
    engine.step([step(slot, prompt[25:])])
    session = engine.decode_session([slot], params(frequency_penalty=0.5), [0], [1])
    said, tokens = [], [7]
    for _ in range(3):
        said += tokens
        tokens = session.step_host(tokens)
    session.set_tokens(tokens)
    for _ in range(2):
        said += tokens
        session.step()
        torch.cuda.synchronize()
        tokens = session.runner.next_tokens[:1].tolist()
    assert_holds(engine, slot, prompt, said)


@pytest.mark.parametrize("rules", [dict(top_p=0.9), dict(logprobs=True), dict(logit_bias={3: 0.5}), dict(repetition_penalty=1.1)])
def test_steps_on_a_guess_are_used(engine, rules, monkeypatch):
    from foundry_b200.engine import engine as module
    made, taken_back, used = [], [], []

    class Session(module.DecodeSession):
        def __init__(self, *args):
            made.append(1)
            super().__init__(*args)

        def cancel_ahead(self):
            taken_back.append(self.has_ahead())
            super().cancel_ahead()

        def _started(self, *args):
            used.append(self.has_ahead())
            return super()._started(*args)

    monkeypatch.setattr(module, "DecodeSession", Session)
    prompts = [tiny.random_tokens(40 + i, 5 + i, engine.spec.vocab_size) for i in range(3)]
    mixed = [params(**rules), params(), params(repetition_penalty=1.2)]
    for sampling in (params(**rules), mixed):
        made.clear(), taken_back.clear(), used.clear()
        engine.generate(prompts, 10, eos_token_id=[], sampling=sampling)
        assert len(made) == 1 and sum(taken_back) == 0
        assert used == [False] + [True] * 8
