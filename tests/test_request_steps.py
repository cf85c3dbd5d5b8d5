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
