"""What the engine makes of requests' own sampling, without a device (tests/stub_engine.py)."""
import numpy as np
import pytest
import torch

import stub_engine
from foundry_b200.engine.context import SequenceStep
from foundry_b200.engine.generate import generate
from foundry_b200.sampling import SamplingParams


@pytest.fixture
def stub(monkeypatch):
    return stub_engine.make(monkeypatch)


def prompt(slot, *tokens):
    return SequenceStep(slot, list(tokens), [len(tokens) - 1])


@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("kind", [list, tuple])
@pytest.mark.parametrize("params", [SamplingParams(), SamplingParams(0.7, 3)])
def test_a_list_of_the_same_plain_parameters(stub, params, kind, rows):
    """One for all rows, whichever way it is given."""
    engine, calls, _ = stub
    prompts = [[1, 2, 3 + i] for i in range(rows)]
    out = generate(engine, prompts, 3, sampling=kind([params] * rows))
    assert out.token_ids == [[7, 8, 9]] * rows
    assert calls == [("select", params)]
    assert stub_engine.Session.made == 1


def test_as_many_parameters_as_rows(stub):
    engine, _, _ = stub
    slots = [engine.open_sequence() for _ in range(2)]
    steps = [prompt(s, 1, 2) for s in slots]
    with pytest.raises(ValueError, match="1 sampling parameters for 2 rows"):
        engine.step_select(steps, [SamplingParams()], [0, 1], [0, 0])


TOP_P, PENALTY = SamplingParams(0.8, 1, top_p=0.9), SamplingParams(0.8, 1, repetition_penalty=1.2)


@pytest.mark.parametrize("sampling", [TOP_P, SamplingParams(logprobs=True), SamplingParams(0.5, 0, top_k=4), PENALTY,
                                      [TOP_P, PENALTY, SamplingParams()], [PENALTY, SamplingParams(logit_bias={3: 1.0}), TOP_P]])
def test_a_step_on_a_guess_is_the_next_step(stub, sampling):
    """Rows with rules, whether they look at a history or not, keep their session, and nothing is taken back."""
    engine, _, _ = stub
    out = generate(engine, [[1, 2], [3, 4], [5, 6, 7]], 9, sampling=sampling)
    assert out.token_ids == [list(range(7, 16))] * 3
    session = stub_engine.Session
    assert (session.made, session.cancelled, session.used) == (1, 0, 7)  # eight steps, the last one of no other


@pytest.mark.parametrize("other", [TOP_P, PENALTY])
def test_a_slot_opened_again_has_a_session_of_its_own(stub, other):
    """Where a row looks at its history, its slot's next sequence starts with an empty one."""
    engine, _, history = stub
    for tokens in ([11, 12], [13, 14]):
        slots = [engine.open_sequence() for _ in range(2)]
        steps = [prompt(slots[0], *tokens), prompt(slots[1], 20)]
        sampling = [PENALTY, other]
        engine.step_select(steps, sampling, [0, 1], [0, 0])
        for count in (1, 2):
            engine.step_select([prompt(s, 7) for s in slots], sampling, [0, 1], [count] * 2, count == 1)
        assert history.rows[slots[0]] == [("prompt", t) for t in tokens] + [("generated", 7)] * 2
        for s in slots:
            engine.close_sequence(s)


def held(history, slot):
    """(the prompt's tokens in the slot's row, the generated ones)"""
    return tuple(sorted(t for w, t in history.rows[slot] if w == what) for what in ("prompt", "generated"))


@pytest.mark.parametrize("pieces", [[[1, 2], [3, 4, 5]], [[1], [2], [3, 4, 5]], [[1, 2, 3, 4], [5]]])
@pytest.mark.parametrize("wants", [False, True])
def test_pieces_of_a_prompt_are_in_the_history(stub, pieces, wants):
    """Whichever step took them: pieces that want nothing, or logits, and single tokens of it."""
    engine, _, history = stub
    for _ in range(2):  # (the slot's next sequence as well)
        slot, other = engine.open_sequence(), engine.open_sequence()
        for piece in pieces[:-1]:
            engine.step([SequenceStep(slot, piece, [len(piece) - 1] if wants else [])])
        engine.step([SequenceStep(other, [50, 51], [])])
        engine.step_select([prompt(slot, *pieces[-1])], PENALTY, [0], [0])
        assert held(history, slot) == ([1, 2, 3, 4, 5], [])
        engine.step_select([prompt(slot, 7)], PENALTY, [0], [1])
        assert held(history, slot) == ([1, 2, 3, 4, 5], [7])
        assert other not in history.rows or not history.rows[other]
        engine.close_sequence(slot)
        engine.close_sequence(other)


@pytest.mark.parametrize("first", [[1, 2, 3], [1]])
@pytest.mark.parametrize("before", [SamplingParams(), SamplingParams(0.8, 1, top_k=9)])
def test_tokens_drawn_without_a_penalty_are_in_the_history(stub, first, before):
    """What a sequence was given and drew before its first penalty, and between two, counts when one comes."""
    engine, _, history = stub
    slot = engine.open_sequence()
    engine.step_select([prompt(slot, *first)], before, [0], [0])
    for count in (1, 2):
        engine.step_select([prompt(slot, 20 + count)], before, [0], [count])
    assert slot not in history.rows
    engine.step_select([prompt(slot, 23)], PENALTY, [0], [3])
    assert held(history, slot) == (first, [21, 22, 23])
    engine.step_select([prompt(slot, 24)], before, [0], [4])
    assert held(history, slot) == (first, [21, 22, 23])
    engine.step_select([prompt(slot, 25, 26)], PENALTY, [0], [5])  # (two tokens of its own at once)
    assert held(history, slot) == (first, [21, 22, 23, 24, 25, 26])
    engine.step([SequenceStep(slot, [30, 31], [])])
    engine.step_select([prompt(slot, 27)], [PENALTY], [0], [7])
    assert held(history, slot) == (first + [30, 31], [21, 22, 23, 24, 25, 26, 27])
    assert engine.tokens_said(slot) == [21, 22, 23, 24, 25, 26, 27]


def test_a_grammar_knows_the_tokens_drawn_before_it(stub):
    engine, _, _ = stub
    slot, asked = engine.open_sequence(), []
    grammar = SamplingParams(allowed_tokens=lambda said: asked.append(list(said)))
    engine.step_select([prompt(slot, 1, 2)], SamplingParams(), [0], [0])
    engine.step_select([prompt(slot, 7)], SamplingParams(), [0], [1])
    engine.step_select([prompt(slot, 8, 9)], grammar, [0], [2])
    assert asked == [[7, 8, 9]]


def test_log_probabilities_are_the_last_steps(stub):
    """A step whose rows ask for none, or that fails, leaves none of an earlier one's."""
    engine, _, _ = stub
    slot = engine.open_sequence()
    engine.step_select([prompt(slot, 1, 2)], SamplingParams(logprobs=True), [0], [0])
    assert engine.last_logprobs() == [-0.5]
    other = engine.open_sequence()
    engine.step_select([prompt(other, 1, 2)], SamplingParams(), [0], [0])
    assert engine.last_logprobs() == []
    engine.step_select([prompt(slot, 7)], SamplingParams(logprobs=True), [0], [1])
    assert engine.last_logprobs() == [-1.0]
    with pytest.raises(ValueError):
        engine.step_select([prompt(slot, 7)], SamplingParams(logit_bias={100: 1.0}), [0], [0])
    assert engine.last_logprobs() == []


@pytest.mark.parametrize("kind", [list, np.array, torch.tensor])
def test_a_callers_tokens_are_its_own_again_behind_the_step(stub, kind):
    engine, _, history = stub
    slot = engine.open_sequence()
    tokens, more = kind([1, 2, 3]), kind([4, 5])
    engine.step([SequenceStep(slot, tokens, [])])
    engine.step_select([SequenceStep(slot, more, [1])], SamplingParams(), [0], [0])
    if kind is list:
        tokens[0] = more[0] = 99
    engine.step_select([prompt(slot, 7)], PENALTY, [0], [1])
    assert held(history, slot) == ([1, 2, 3, 4, 5], [7])
