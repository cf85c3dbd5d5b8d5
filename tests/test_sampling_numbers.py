"""Sampling parameters are numbers that the kernels' 32 bits hold."""
import math

import numpy as np
import pytest

from foundry_b200.sampling import SamplingParams
from foundry_b200.sampling.rules import RowRules

LARGEST = float(np.finfo(np.float32).max)


@pytest.mark.parametrize("wrong", [
    dict(repetition_penalty=1e39), dict(repetition_penalty=1e-46), dict(frequency_penalty=1e39), dict(frequency_penalty=-1e39),
    dict(presence_penalty=4e38), dict(logit_bias={3: 1e39}), dict(logit_bias={3: -1e39}), dict(top_k=math.inf), dict(top_k=math.nan),
    dict(top_k=2.5), dict(temperature=math.nan)])
def test_what_32_bits_do_not_hold_is_refused(wrong):
    """A bias of 1e39 would be infinity there, a repetition penalty of 1e-46 a division by zero."""
    with pytest.raises(ValueError, match=next(iter(wrong))):
        SamplingParams(**wrong)


def test_what_they_hold_reaches_the_kernels():
    p = SamplingParams(0.5, top_k=3.0, top_p=1e-30, min_p=1e-30, repetition_penalty=1e-30, frequency_penalty=LARGEST,
                       presence_penalty=-LARGEST, logit_bias={0: LARGEST, 5: -LARGEST, 7: -math.inf})
    rules = RowRules(1, 10, "cpu", bias_room=64)
    with np.errstate(all="raise"):
        rules.fill([p], [-1])
    assert np.array_equal(rules.edits.bias.values[:3].numpy(), np.array([LARGEST, -LARGEST, -np.inf], np.float32))
    assert float(rules.rules.top_p[0]) > 0 and float(rules.rules.min_p[0]) > 0 and int(rules.rules.top_k[0]) == 3
