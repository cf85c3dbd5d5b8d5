"""How the next token is chosen.

The reference chooses greedily and in no other way: argmax over the
vocabulary, the lowest index among equal logits (src/generate/mod.rs:192-204,
src/metal/kernels/reduce.metal:67-68). `temperature = 0` is that rule.
A positive temperature samples from softmax(logits / temperature); the draw is
a pure function of (seed, request index, number of tokens the request has
generated), so a request's tokens do not depend on its batch.

Further rules are a request's own, each off by default:

  on the logits, in this order (csrc/logit_edits.cuh): `repetition_penalty` r (a token that the
    prompt holds or that was generated: v / r where v > 0, else v * r), `frequency_penalty` f and
    `presence_penalty` p (generated c > 0 times: v - f c - p), `logit_bias` {token: b} (v + b; -inf
    bans a token), `allowed_tokens` (a grammar: called with the tokens generated so far, it says
    which may come next, or None for all)
  on the draw, in this order (csrc/sample_rules.cu): `top_k` most likely tokens, of these the fewest
    whose probability reaches `top_p`, of these the ones at least `min_p` times as likely as the first

`logprobs` asks for each token's log-probability: under softmax(edited logits / temperature) (greedy: of
the edited logits), before the draw's rules cut anything off.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable, Iterable, Mapping, Optional, Sequence, Tuple, Union

LARGEST = float.fromhex("0x1.fffffep127")  # of 32 bits
SMALLEST_TEMPERATURE, SMALLEST_PENALTY = 2.0 ** -120, 2.0 ** -126  # csrc/sample_rules.cu; not rounded to zero

Allowed = Callable[[Sequence[int]], Optional[Iterable[int]]]


@dataclass(frozen=True)
class SamplingParams:
    temperature: float = 0.0
    seed: int = 0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    repetition_penalty: float = 1.0
    frequency_penalty: float = 0.0
    presence_penalty: float = 0.0
    logit_bias: Union[Mapping[int, float], Tuple[Tuple[int, float], ...]] = ()
    allowed_tokens: Optional[Allowed] = None
    logprobs: bool = False

    def __post_init__(self):
        if not (self.temperature >= 0.0):
            raise ValueError(f"temperature must not be negative, got {self.temperature}")
        if not 0 <= self.top_k < 1 << 31 or int(self.top_k) != self.top_k:
            raise ValueError(f"top_k must be a whole number of tokens or 0, got {self.top_k}")
        if not 0.0 < self.top_p <= 1.0:
            raise ValueError(f"top_p must lie in (0, 1], got {self.top_p}")
        if not 0.0 <= self.min_p <= 1.0:
            raise ValueError(f"min_p must lie in [0, 1], got {self.min_p}")
        # (the kernels' numbers are of 32 bits: what is finite in 64 may be infinite there, or zero)
        if not SMALLEST_PENALTY <= self.repetition_penalty <= LARGEST:
            raise ValueError(f"repetition_penalty must be positive and finite in 32 bits, got {self.repetition_penalty}")
        for name in ("frequency_penalty", "presence_penalty"):
            if not abs(getattr(self, name)) <= LARGEST:
                raise ValueError(f"{name} must be finite in 32 bits, got {getattr(self, name)}")
        pairs = self.logit_bias.items() if isinstance(self.logit_bias, Mapping) else self.logit_bias
        pairs = tuple(sorted((int(t), float(b)) for t, b in pairs))
        if len({t for t, _ in pairs}) != len(pairs) or any(t < 0 for t, _ in pairs):
            raise ValueError("logit_bias names a token twice, or a negative one")
        if not all(abs(b) <= LARGEST or b == -math.inf for _, b in pairs):
            raise ValueError("logit_bias values are finite in 32 bits, or -inf")
        object.__setattr__(self, "logit_bias", pairs)

    @property
    def greedy(self) -> bool:
        return self.temperature == 0.0

    @property
    def held_temperature(self) -> float:
        """The temperature as the kernels calculate with it (32 bits would make zero, the greedy choice, of the
        smallest ones)."""
        return min(max(self.temperature, SMALLEST_TEMPERATURE), LARGEST) if self.temperature else 0.0

    @property
    def needs_history(self) -> bool:
        """Whether the draw depends on which tokens the sequence holds."""
        return (self.repetition_penalty != 1.0 or self.frequency_penalty != 0.0
                or self.presence_penalty != 0.0)

    @property
    def plain(self) -> bool:
        """Temperature and seed say all there is to say."""
        return not (self.top_k or self.top_p < 1.0 or self.min_p or self.needs_history
                    or self.logit_bias or self.allowed_tokens is not None or self.logprobs)


def params_of_rows(params, n: int):
    """One `SamplingParams` a row: of one for all, or of a sequence."""
    if isinstance(params, SamplingParams):
        return [params] * n
    rows = list(params)
    if len(rows) != n:
        raise ValueError(f"{len(rows)} sampling parameters for {n} rows")
    return rows


def is_ruled(params) -> bool:
    """Whether rows need more than one temperature for all (a single plain `SamplingParams`, or the
    same one for every row, does not)."""
    if isinstance(params, SamplingParams):
        return not params.plain
    rows = list(params)
    return any(not p.plain for p in rows) or any(p != rows[0] for p in rows[1:])
