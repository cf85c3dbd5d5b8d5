"""The uniform numbers behind a draw lie below one, also the largest: a token whose number's 24 bits are all set has
large noise, not infinite noise, by which it would win whatever its logit."""
import numpy as np
import pytest
import torch

from foundry_b200.sampling import gumbel_scores, stream_key, uniform24

MASK = (1 << 64) - 1
GOLDEN, M1, M2 = 0x9e3779b97f4a7c15, 0xbf58476d1ce4e5b9, 0x94d049bb133111eb


def unmixed(z):
    """The number whose mix64 is z: each step of it can be undone."""
    def unshifted(y, s):
        x = y
        for _ in range(64 // s + 1):
            x = y ^ (x >> s)
        return x
    z = (unshifted(z, 31) * pow(M2, -1, 1 << 64)) & MASK
    z = (unshifted(z, 27) * pow(M1, -1, 1 << 64)) & MASK
    return unshifted(z, 30)


def stream_of(step, token):
    """A random stream in which all 64 bits of this token's number are set at this step."""
    z = (unmixed(MASK) - GOLDEN * (token + 1)) & MASK
    stream = (unmixed(z) - GOLDEN * (step + 1)) & MASK
    return stream - (1 << 64) if stream >> 63 else stream


def seed_of(stream, key):
    return (unmixed(stream & MASK) - GOLDEN * (key + 1)) & MASK


@pytest.mark.parametrize("step,token", [(0, 0), (7, 11), (1000, 63)])
def test_the_largest_number_on_the_host(step, token):
    stream = stream_of(step, token)
    seed = seed_of(stream, 3)
    assert stream_key(seed, 3) == stream
    u = uniform24(seed, 3, step, 64)
    assert u[token] == np.float32(1 - 2.0 ** -24) and (u < 1).all() and (u > 0).all()
    logits = np.zeros(64, np.float32)
    logits[5] = 40.0
    scores = gumbel_scores(logits, 1.0, seed, 3, step)
    assert np.isfinite(scores).all() and int(np.argmax(scores)) == 5


@pytest.mark.gpu
@pytest.mark.parametrize("V", [64, 5001, 128256])
def test_the_largest_number_wins_nothing_by_itself(V):
    """-log(-log(1 - 2^-24)) is 16.6: enough against 16 and not against 17.5."""
    from foundry_b200.kernels import ops
    where = [11, 0, V - 1]
    logits = torch.full((3, V), -100.0, device="cuda:0")
    logits[0, 5], logits[0, 11] = 17.5, 0.0
    logits[1, V - 1], logits[1, 0] = 40.0, 0.0
    logits[2, 7], logits[2, V - 1] = 10.0, 0.0
    steps = [0, 3, 9]
    streams = [stream_of(s, t) for s, t in zip(steps, where)]
    for t, s, k in zip(where, steps, streams):  # (the other one's noise is between -2.9 and 10)
        assert uniform24(seed_of(k, 0), 0, s, V)[t] == np.float32(1 - 2.0 ** -24)
    got = ops.select_tokens(logits, torch.empty(3, dtype=torch.int32, device="cuda:0"), torch.ones(3, device="cuda:0"),
                            torch.tensor(streams, device="cuda:0"), torch.tensor(steps, device="cuda:0"))
    host = logits.cpu().numpy()
    want = [int(np.argmax(gumbel_scores(host[r], 1.0, seed_of(streams[r], 0), 0, steps[r]))) for r in range(3)]
    assert got.tolist() == want and want[1] == V - 1
    again, _ = ops.sample_tokens(logits, ops.SampleRules(torch.ones(3, device="cuda:0"), streams=torch.tensor(streams, device="cuda:0"),
                                                         steps=torch.tensor(steps, device="cuda:0")))
    assert again.tolist() == want
