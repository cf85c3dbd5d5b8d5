"""Steps of no rows, with every kind of edit that rows may bring."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from foundry_b200.kernels import ops
    return ops


def test_no_rows_with_every_edit(ops):
    V = 70
    none = lambda dtype: torch.empty(0, dtype=dtype, device=DEV)  # noqa: E731
    history = ops.TokenHistory.empty(3, V, DEV)
    edits = ops.LogitEdits(history, none(torch.int32), none(torch.float32), none(torch.float32), none(torch.float32),
                           ops.TokenBiases.from_rows([], DEV), torch.zeros(2, 3, dtype=torch.int32, device=DEV), none(torch.int32))
    logits = torch.empty(0, V, device=DEV)
    assert ops.edit_logits(logits, edits).shape == (0, V)
    tokens, logprobs = ops.sample_tokens(logits, ops.SampleRules(none(torch.float32)), edits, record=none(torch.int32))
    assert tokens.shape == logprobs.shape == (0,)
    ops.record_tokens(history, none(torch.int32), none(torch.int32))
    assert not history.counts.any()


def test_rows_with_biases_for_none_of_them(ops):
    logits = torch.randn(3, 70, device=DEV)
    edits = ops.LogitEdits(bias=ops.TokenBiases.from_rows([None, {}, None], DEV))
    assert torch.equal(ops.edit_logits(logits, edits), logits)
    assert torch.equal(ops.sample_tokens(logits, ops.SampleRules(), edits)[0].long(), logits.argmax(1))
