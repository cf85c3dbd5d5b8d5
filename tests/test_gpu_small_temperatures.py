"""Temperatures near zero and near the largest number: the draw goes over into the largest logit and into equal
shares, and every log-probability stays one."""
import numpy as np
import pytest
import torch

import plain_requests as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
SMALL = [1e-3, 1e-20, 2e-37, 9.3e-38, 5e-38, 1.1e-38, 2.9e-39, 1e-39, 1e-45]
RULES = [dict(), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=3, top_p=0.5, min_p=0.01)]


@pytest.fixture(scope="module")
def ops():
    from foundry_b200.kernels import ops
    return ops


def drawn(ops, logits, temperature, top_k=0, top_p=1.0, min_p=0.0):
    n = logits.shape[0]
    tokens, logprobs = ops.sample_tokens(logits, ops.SampleRules(
        torch.tensor([temperature] * n, dtype=torch.float32, device=DEV), torch.full((n,), top_k, dtype=torch.int32, device=DEV),
        torch.full((n,), top_p, device=DEV), torch.full((n,), min_p, device=DEV), torch.arange(n, device=DEV),
        torch.arange(n, device=DEV)))
    return tokens.tolist(), logprobs.tolist()


@pytest.mark.parametrize("rules", RULES)
@pytest.mark.parametrize("temperature", SMALL)
@pytest.mark.parametrize("n,V", [(3, 1000), (2, 128256)])
def test_small_ones_take_the_largest_logit(ops, n, V, temperature, rules):
    """Its lead over the second one is half a unit and more: 500 temperatures at least, so that its share is one."""
    logits = torch.randn(n, V, generator=torch.Generator().manual_seed(V)).to(DEV).clamp(max=5.0)
    where = [7, V - 1, V // 2][:n]
    for r, t in enumerate(where):
        logits[r, t] = 5.5
    tokens, logprobs = drawn(ops, logits, temperature, **rules)
    assert tokens == where and logprobs == [0.0] * n


@pytest.mark.parametrize("rules", RULES)
@pytest.mark.parametrize("temperature", SMALL[1:])
def test_small_ones_share_among_equals(ops, temperature, rules):
    logits = torch.randn(64, 3000, generator=torch.Generator().manual_seed(1)).to(DEV)
    logits[:, [4, 2999]] = 9.0
    tokens, logprobs = drawn(ops, logits, temperature, **rules)
    # (either one of both; where the rules leave the first half of the weight, the first)
    if rules.get("top_p", 1.0) > 0.5:
        assert set(tokens) == {4, 2999} and 10 < tokens.count(4) < 54
    else:
        assert set(tokens) == {4}
    assert logprobs == [float(np.float32(np.log(0.5)))] * 64


@pytest.mark.parametrize("temperature", SMALL)
@pytest.mark.parametrize("V", [1000, 128256])
def test_small_ones_in_the_plain_selection(ops, V, temperature):
    """Logits of some hundreds too: none of them over a temperature is infinite."""
    logits = torch.randn(4, V, generator=torch.Generator().manual_seed(V)).to(DEV)
    logits[0, 9], logits[0, 3] = 700.0, 600.0
    logits[1, 9], logits[1, 3] = 0.0, -1.0
    logits[1] -= 50.0
    logits[1, 9] = 0.0
    logits[2] = -300.0 - logits[2].abs()
    logits[2, V - 1] = -290.0
    logits[3, 5] = 30.0
    got = ops.select_tokens(logits, torch.empty(4, dtype=torch.int32, device=DEV),
                            torch.tensor([temperature] * 4, dtype=torch.float32, device=DEV),
                            torch.arange(4, device=DEV), torch.arange(4, device=DEV))
    assert got.tolist() == [9, 9, V - 1, 5]


@pytest.mark.parametrize("temperature", [1e30, 3.4e38, float("inf")])
def test_large_ones_give_equal_shares(ops, temperature):
    n, V = 200, 40
    logits = torch.randn(n, V, generator=torch.Generator().manual_seed(2)).to(DEV)
    logits[:, 1] = float("-inf")
    heat = torch.full((n,), temperature, device=DEV)
    some = torch.arange(n, device=DEV)
    tokens = ops.select_tokens(logits, torch.empty(n, dtype=torch.int32, device=DEV), heat, some, some)
    again, logprobs = ops.sample_tokens(logits, ops.SampleRules(heat, streams=some, steps=some))
    assert torch.equal(tokens, again)
    want = [int(np.argmax(np.where(np.arange(V) == 1, -np.inf, plain.noise(r, r, V)))) for r in range(n)]
    assert tokens.tolist() == want
    assert np.allclose(logprobs.cpu().numpy(), -np.log(39.0), rtol=2.0 ** -22)


@pytest.mark.parametrize("temperature", [float("nan"), -1.0, 0.0])
def test_no_temperature_is_the_largest_logit(ops, temperature):
    logits = torch.randn(5, 300, generator=torch.Generator().manual_seed(2)).to(DEV)
    heat, some = torch.full((5,), temperature, device=DEV), torch.arange(5, device=DEV)
    tokens = ops.select_tokens(logits, torch.empty(5, dtype=torch.int32, device=DEV), heat, some, some)
    again, logprobs = ops.sample_tokens(logits, ops.SampleRules(heat, streams=some, steps=some))
    assert tokens.tolist() == again.tolist() == logits.argmax(1).tolist()
    assert torch.allclose(logprobs, torch.log_softmax(logits, 1).max(1).values, rtol=1e-5)
