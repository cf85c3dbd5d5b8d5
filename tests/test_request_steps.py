"""What the engine makes of requests' own sampling, without a device (tests/stub_engine.py)."""
import pytest

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
        assert history.rows[slots[0]] == [("prompt", t) for t in tokens]
        for s in slots:
            engine.close_sequence(s)
