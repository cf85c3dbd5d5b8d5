"""The rows of a step whose requests bring rules of their own, as the kernels take them.

`RowRules` holds the device tensors of `ops.SampleRules` and `ops.LogitEdits` for a number of rows, the
host copies beside them, and what sends one to the other: a ring of pinned buffers where steps are queued
ahead of the device (`StagingRing`; the tensors then stay where they are, as a captured step needs), or a
plain copy for a single step.
"""
from __future__ import annotations

from typing import Iterable, List, Optional, Sequence

import numpy as np
import torch

from ..kernels import ops
from .params import SamplingParams

BIAS_ROOM = 64  # entries that a step of a few biases has room for; more go in powers of two


def bias_room(params: Sequence[SamplingParams]) -> int:
    count = sum(len(p.logit_bias) for p in params)
    room = BIAS_ROOM if count else 0
    while room < count:
        room *= 2
    return room


def check_vocabulary(params: Sequence[SamplingParams], vocab: int) -> None:
    for p in params:
        if p.logit_bias and p.logit_bias[-1][0] >= vocab:
            raise ValueError(f"logit_bias names token {p.logit_bias[-1][0]}, outside the vocabulary of {vocab}")


def mask_bits(allowed: Iterable[int], vocab: int) -> np.ndarray:
    """The bits of a mask that allows these tokens, int32 words."""
    ids = np.fromiter((int(t) for t in allowed), dtype=np.int64)
    if ids.size and not (0 <= ids.min() and ids.max() < vocab):
        raise ValueError(f"allowed_tokens names a token outside the vocabulary of {vocab}")
    flags = np.zeros((vocab + 31) // 32 * 32, np.uint8)
    flags[ids] = 1
    return np.packbits(flags, bitorder="little").view(np.int32)


def masks_of(params: Sequence[SamplingParams], said: Sequence[Sequence[int]], vocab: int):
    """The bits of what each row's grammar allows behind these tokens of its own, or None: all."""
    masks = []
    for p, tokens in zip(params, said):
        allowed = None if p.allowed_tokens is None else p.allowed_tokens(tokens)
        masks.append(None if allowed is None else mask_bits(allowed, vocab))
    return masks


class _Copied:
    """A `StagingRing`'s interface for values that are sent once."""

    def __init__(self, count: int, dtype: torch.dtype, device):
        self.dev = torch.zeros(count, dtype=dtype, device=device)
        self._host = torch.zeros(count, dtype=dtype)
        self.values = self._host.numpy()

    def upload(self) -> int:
        self.dev.copy_(self._host)
        return self._host.numel() * self._host.element_size()


class RowRules:
    def __init__(self, rows: int, vocab: int, device, history: Optional[ops.TokenHistory] = None,
                 bias_room: int = 0, masks: bool = False, ahead: bool = False):
        if ahead:
            from ..engine.staging import StagingRing as Ring
        else:
            Ring = _Copied
        self.rows, self.vocab, self.bias_room = rows, vocab, bias_room
        b, room = rows, bias_room
        # one int32 and one float32 upload: top_k | history rows | mask rows | bias starts | bias ids,
        # temperature | top_p | min_p | three penalties | bias values
        self.ints = Ring(3 * b + b + 1 + room, torch.int32, device)
        self.floats = Ring(6 * b + room, torch.float32, device)
        self.meta = Ring(2 * b, torch.int64, device)  # random streams | tokens generated
        words = (vocab + 31) // 32
        self.bits = Ring(b * words, torch.int32, device) if masks else None
        i, f, m = self.ints.dev, self.floats.dev, self.meta.dev
        self.rules = ops.SampleRules(f[:b], i[:b], f[b:2 * b], f[2 * b:3 * b], m[:b], m[b:])
        given = {}
        if history is not None:
            given.update(history=history, history_rows=i[b:2 * b], repetition=f[3 * b:4 * b],
                         frequency=f[4 * b:5 * b], presence=f[5 * b:6 * b])
        if room:
            given["bias"] = ops.TokenBiases(i[3 * b:4 * b + 1], i[4 * b + 1:], f[6 * b:])
        if masks:
            given.update(allowed=self.bits.dev.view(b, words), allowed_rows=i[2 * b:3 * b])
        self.edits = ops.LogitEdits(**given)
        self.logprobs = torch.zeros(b, dtype=torch.float32, device=device)

    def fill(self, params: Sequence[SamplingParams], history_rows: Sequence[int]) -> int:
        """The rules of the first rows (the others draw greedily from unedited logits); returns the
        bytes sent."""
        b, n, i, f = self.rows, len(params), self.ints.values, self.floats.values
        i[:] = 0
        f[:] = 0.0
        i[:n] = [min(p.top_k, self.vocab) for p in params]
        i[b:3 * b] = -1
        i[b:b + n] = history_rows
        f[:n] = [p.held_temperature for p in params]
        f[b:2 * b] = 1.0
        f[b:b + n] = [p.top_p for p in params]
        f[2 * b:2 * b + n] = [p.min_p for p in params]
        f[3 * b:4 * b] = 1.0
        f[3 * b:3 * b + n] = [p.repetition_penalty for p in params]
        f[4 * b:4 * b + n] = [p.frequency_penalty for p in params]
        f[5 * b:5 * b + n] = [p.presence_penalty for p in params]
        if self.bias_room:
            starts = np.zeros(b + 1, np.int32)
            starts[1:n + 1] = np.cumsum([len(p.logit_bias) for p in params])
            starts[n + 1:] = starts[n]
            i[3 * b:4 * b + 1] = starts
            entries = [e for p in params for e in p.logit_bias]
            i[4 * b + 1:4 * b + 1 + len(entries)] = [t for t, _ in entries]
            f[6 * b:6 * b + len(entries)] = [v for _, v in entries]
        return self.ints.upload() + self.floats.upload()

    def set_steps(self, streams: Sequence[int], counts: Sequence[int]) -> int:
        b, n, m = self.rows, len(streams), self.meta.values
        m[:n] = streams
        m[b:b + n] = counts
        return self.meta.upload()

    def set_masks(self, masks: Sequence[Optional[np.ndarray]]) -> int:
        """Which tokens each row allows, as `masks_of` gives them."""
        b, words = self.rows, (self.vocab + 31) // 32
        bits, where = self.bits.values.reshape(b, words), self.ints.values
        where[2 * b:3 * b] = -1
        for r, mask in enumerate(masks):
            if mask is not None:
                bits[r] = mask
                where[2 * b + r] = r
        return self.bits.upload() + self.ints.upload()

    def draw(self, logits: torch.Tensor, out: torch.Tensor, record: Optional[torch.Tensor] = None,
             also: Optional[torch.Tensor] = None):
        return ops.sample_tokens(logits, self.rules, self.edits, out=out, logprobs=self.logprobs,
                                 record=None if self.edits.history is None else record, also=also)
