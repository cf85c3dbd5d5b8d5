"""An `Engine` without a device: its own bookkeeping of requests, with the model, the cache and the sessions replaced."""
import types

import torch

from foundry_b200.engine import engine as module
from foundry_b200.engine.decode import DecodeSession
from foundry_b200.engine.engine import Engine
from foundry_b200.kernels import ops
from foundry_b200.sampling import is_ruled, params_of_rows


class Slots:
    def __init__(self, count):
        self.open, self.count = set(), count

    @property
    def free(self):
        return self.count - len(self.open)

    def is_held(self, slot):
        return slot in self.open


class Cache:
    scratch_slot, max_tokens = 8, 4096

    def free_tokens(self):
        return self.max_tokens

    def __init__(self):
        self.table = types.SimpleNamespace(slots=Slots(8))

    def open_sequence(self):
        slot = min(set(range(8)) - self.table.slots.open)
        self.table.slots.open.add(slot)
        return slot

    def close_sequence(self, slot):
        self.table.slots.open.remove(slot)

    def step_token_limit(self):
        return None


class Session:
    """As `DecodeSession`, with steps that are counted and started on a guess whenever they may be."""
    made, cancelled, used = 0, 0, 0
    _note = DecodeSession._note

    def step_logits(self, tokens):
        self._note(tokens, prompt=True)
        return torch.zeros(len(tokens), 100)

    def __init__(self, engine, slots, sampling, keys=None, counts=None):
        type(self).made += 1
        self.engine, self.slots, self.keys = engine, list(slots), list(keys)
        self.sampling = sampling if not isinstance(sampling, (list, tuple)) else list(sampling)
        self.params = params_of_rows(sampling, len(self.slots))
        self.rules = (0, False, False) if is_ruled(self.sampling) else None
        self.history_rows = [s if self.rules and p.needs_history else -1
                             for s, p in zip(self.slots, self.params)]
        self.adapters = engine.adapters_of(self.slots)
        self.last_logprobs, self.ahead = [], False
        engine.complete_history([r for r in self.history_rows if r >= 0])

    def cancel_ahead(self):
        type(self).cancelled += self.ahead
        self.ahead = False

    def step_host(self, tokens, more=False, counts=None):
        type(self).used += self.ahead
        self.ahead = more
        said = [(r, t) for r, t in zip(self.history_rows, tokens) if r >= 0]
        self.engine.complete_history([r for r, _ in said])
        for r, t in said:
            self.engine._history.rows[r].append(("generated", t))
        self._note(tokens)
        self.last_logprobs = [-1.0] * len(tokens)
        return [t + 1 for t in tokens]


class History:
    """What is recorded, by row: {row: [(what, token)]}."""

    def __init__(self):
        self.rows = {}

    def clear(self, rows):
        for r in rows:
            self.rows[r] = []


def make(monkeypatch):
    """(engine, its sampler's calls, its history): steps give logits of zeros, draws token 7."""
    engine = Engine.__new__(Engine)
    engine.spec = types.SimpleNamespace(vocab_size=100, eos_token_ids=(), max_positions=1000)
    engine.device, engine.cache = torch.device("cpu"), Cache()
    for name, value in dict(_session=None, _history=History(), _unread=set(), _told={}, _last_logprobs=[],
                            adapters=None, _adapter_of={}, _runners={}, scratch=("test", 0), use_graphs=False,
                            _prompts=types.SimpleNamespace(wants=lambda steps: True, step=lambda steps: torch.zeros(
                                sum(len(s.want) for s in steps), 100))).items():
        setattr(engine, name, value)
    calls = []

    class Sampler:
        def select(self, logits, params, keys=None, steps=None):
            calls.append(("select", params))
            params.greedy  # (one for all rows)
            return torch.full((logits.shape[0],), 7, dtype=torch.int32)

        def draw(self, logits, params, keys, steps, history, rows, masks):
            calls.append(("draw", params, rows, masks))
            n = logits.shape[0]
            return torch.full((n,), 7, dtype=torch.int32), torch.full((n,), -0.5)

    def record(history, rows, tokens, what="generated"):
        for r, t in zip(rows.tolist(), tokens.tolist()):
            history.rows[r].append((what, t))

    engine.sampler = Sampler()
    Session.made = Session.cancelled = Session.used = 0
    monkeypatch.setattr(module, "DecodeSession", Session)
    monkeypatch.setattr(ops, "wait_for_stream", lambda: None)
    monkeypatch.setattr(ops, "raise_on_device_failure", lambda: None)
    monkeypatch.setattr(ops, "record_tokens", record)
    return engine, calls, engine._history
