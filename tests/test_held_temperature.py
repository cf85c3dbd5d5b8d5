"""A temperature as the kernels hold it (tests/test_gpu_small_temperatures.py has the draws)."""
import numpy as np
import pytest

from foundry_b200.sampling import SamplingParams, gumbel_scores
from foundry_b200.sampling.rules import RowRules


@pytest.mark.parametrize("given,held", [(0.0, 0.0), (0.7, 0.7), (1e-50, 2.0 ** -120), (1e-45, 2.0 ** -120), (5e-324, 2.0 ** -120),
                                        (2e-36, 2e-36), (1e39, 2.0 ** 128 - 2.0 ** 104), (float("inf"), 2.0 ** 128 - 2.0 ** 104)])
def test_temperatures(given, held):
    """Every positive one stays one in 32 bits: it is no greedy row, whose log-probabilities are those of T = 1."""
    params = SamplingParams(given)
    assert params.held_temperature == held
    assert (np.float32(held) > 0) == (given > 0) and np.isfinite(np.float32(held))
    rules = RowRules(2, 40, "cpu")
    with np.errstate(over="raise"):
        rules.fill([params, SamplingParams()], [-1, -1])
    assert rules.rules.temperature.tolist() == [float(np.float32(held)), 0.0]


@pytest.mark.parametrize("temperature", [1e-50, 1e-38, 1e-3])
def test_the_host_restatement_of_small_ones(temperature):
    logits = np.array([600.0, 0.0, 700.0, -700.0], np.float32)
    scores = gumbel_scores(logits, temperature, 1, 2, 3)
    assert np.isfinite(scores).all() and int(np.argmax(scores)) == 2
