"""How near a drawn token's log-probability is to the exact one."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("rules", [dict(), dict(top_k=60), dict(top_p=0.9999)])
@pytest.mark.parametrize("temperature", [0.7, 1.0, 1.3])
def test_tokens_far_from_the_best_one(temperature, rules):
    """The token's own lead is of 64 bits, the sum of the weights is as near as its weights are: the best one's is
    one exactly, another's off by 2^-24 (3 |z| + 4) of itself (the difference, the factor and their product are rounded,
    the power of two is within 2^-22). Then one rounding."""
    from foundry_b200.kernels import ops
    n, V = 6000, 64
    g = torch.Generator().manual_seed(int(temperature * 10))
    logits = (torch.randn(n, V, generator=g) * 0.3 - 7.5 * temperature).float()
    logits[:, 17] = torch.rand(n, generator=g) * 0.1
    some = torch.arange(n, device=DEV)
    tokens, logprobs = ops.sample_tokens(logits.to(DEV), ops.SampleRules(
        torch.full((n,), temperature, device=DEV), torch.full((n,), rules.get("top_k", 0), dtype=torch.int32, device=DEV),
        torch.full((n,), rules.get("top_p", 1.0), device=DEV), streams=some, steps=some))
    tokens, logprobs = tokens.long().cpu().numpy(), logprobs.double().cpu().numpy()
    far = np.nonzero(tokens != 17)[0]
    assert len(far) > 100
    v = logits.double().numpy()
    z = (v - v.max(1, keepdims=True)) / float(np.float32(temperature))
    w = np.exp(z)
    want = z[np.arange(n), tokens] - np.log(w.sum(1))
    others = np.where(z < 0, w * (3 * np.abs(z) + 4), 0.0).sum(1) / w.sum(1)
    off = np.abs(logprobs - want)
    assert (off <= 2.0 ** -24 * (np.abs(want) + others)).all(), (off / (2.0 ** -24 * (np.abs(want) + others))).max()
