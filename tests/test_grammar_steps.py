"""A grammar is asked before a step changes anything, and a step that was refused may come again, without a device."""
import types

import numpy as np
import pytest
import torch

import stub_engine
from foundry_b200.cache.pages import CacheFull
from foundry_b200.engine.context import SequenceStep
from foundry_b200.engine.decode import DecodeSession
from foundry_b200.kernels import ops
from foundry_b200.sampling import SamplingParams


class Grammar:
    """Keeps what it was asked (its own copy of it), allows what it is told to."""

    def __init__(self, allowed=(1, 2)):
        self.asked, self.allowed = [], allowed

    def __call__(self, said):
        self.asked.append(list(said))
        said.append(-1)  # (the list is the callback's own)
        if isinstance(self.allowed, Exception):
            raise self.allowed
        return self.allowed


class Ring:
    def upload(self, start=0):
        return 0


class Rules:
    def __init__(self):
        self.masks, self.logprobs = [], torch.zeros(1)

    def fill(self, *args):
        return 0

    def set_steps(self, *args):
        return 0

    def set_masks(self, masks):
        self.masks.append([None if m is None else np.unpackbits(m.view(np.uint8), bitorder="little").nonzero()[0].tolist()
                           for m in masks])
        return 0


@pytest.fixture
def session(monkeypatch):
    """A session of one row whose steps run nowhere; `session.full` refuses the next one for want of room."""
    engine, _, _ = stub_engine.make(monkeypatch)
    slot = engine.open_sequence()
    made = DecodeSession.__new__(DecodeSession)
    grammar = Grammar()
    runner = types.SimpleNamespace(
        rules=Rules(), rules_of=None, fields=Ring(), meta_start=1, bucket=1, host_np=np.zeros(1, np.int32), ran=0,
        tokens_host=torch.zeros(1, dtype=torch.int32), next_tokens=torch.tensor([2], dtype=torch.int32), logprobs_host=torch.zeros(1))

    def run():
        runner.ran += 1
    runner.run = run

    def prepare():
        if made.full:
            made.full = False
            raise CacheFull("no room")
        engine.cache.table.length[slot] += 1
        return runner

    engine.cache.table.length = {slot: 5}
    for name, value in dict(engine=engine, slots=[slot], params=[SamplingParams(allowed_tokens=grammar)], streams=[0], counts=[1],
                            rules=(0, True, False), history_rows=[-1], said_rows=[], _ahead=None, full=False, runner=runner, _prepare=prepare,
                            _read=types.SimpleNamespace(record=lambda: None, synchronize=lambda: None)).items():
        setattr(made, name, value)
    monkeypatch.setattr(ops, "raise_on_device_failure", lambda: None)
    return made, grammar, runner


def test_a_refused_step_comes_again(session):
    made, grammar, runner = session
    made.step_host([4], counts=[1])
    made.full = True
    with pytest.raises(CacheFull):
        made.step_host([5], counts=[2])
    made.step_host([5], counts=[2])
    made.step_host([6], counts=[3])
    assert grammar.asked == [[4], [4, 5], [4, 5], [4, 5, 6]]
    assert runner.ran == 3 and made.engine.cache.table.length == {0: 8}
    assert made.engine.tokens_said(0) == [4, 5, 6]


@pytest.mark.parametrize("wrong", [RuntimeError("no such state"), [3, 100]])
def test_a_grammar_that_fails_leaves_the_sequence_as_it_was(session, wrong):
    made, grammar, runner = session
    made.step_host([4], counts=[1])
    good, grammar.allowed = grammar.allowed, wrong
    with pytest.raises(RuntimeError if isinstance(wrong, Exception) else ValueError):
        made.step_host([5], counts=[2])
    assert runner.ran == 1 and made.engine.cache.table.length == {0: 6}
    grammar.allowed = good
    made.step_host([5], counts=[2])
    assert grammar.asked == [[4], [4, 5], [4, 5]] and runner.rules.masks == [[[1, 2]]] * 2
    assert made.engine.tokens_said(0) == [4, 5]


@pytest.mark.parametrize("wrong", [dict(allowed_tokens=Grammar(RuntimeError("no such state"))), dict(allowed_tokens=Grammar([100])),
                                   dict(logit_bias={100: 1.0})])
@pytest.mark.parametrize("count", [0, 2])
def test_a_refused_prompt_was_not_run(monkeypatch, wrong, count):
    engine, calls, _ = stub_engine.make(monkeypatch)
    slot, ran = engine.open_sequence(), []
    run = engine._prompts.step
    engine._prompts.step = lambda steps: ran.append(steps) or run(steps)
    step = [SequenceStep(slot, [1, 2, 3], [2])]
    with pytest.raises((RuntimeError, ValueError)):
        engine.step_select(step, [SamplingParams(**wrong)], [0], [count])
    assert not ran and not calls and engine.tokens_said(slot) == []
    grammar = Grammar()
    engine.step_select(step, [SamplingParams(allowed_tokens=grammar)], [0], [count])
    assert len(ran) == 1 and grammar.asked == [[1, 2, 3] if count else []]
    assert engine.tokens_said(slot) == ([1, 2, 3] if count else [])
