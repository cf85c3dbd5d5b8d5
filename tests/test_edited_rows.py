"""Where edited logits may go: into rows of their own, or into the logits' place, not into a part of it."""
import pytest
import torch

from foundry_b200.kernels import ops


@pytest.mark.parametrize("n", [1, 2, 5])
@pytest.mark.parametrize("stride,other_stride", [(10, 10), (25, 25), (25, 10), (10, 30)])
@pytest.mark.parametrize("shift", [-60, -25, -20, -15, -10, -9, -1, 0, 1, 9, 10, 11, 15, 16, 24, 25, 26, 49, 50, 200])
def test_rows_that_are_partly_the_same(n, stride, other_stride, shift):
    """Against the sets of their elements; rows of different strides count as such wherever their ranges meet."""
    width, one = 10, 1000
    mine = [one + r * stride + i for r in range(n) for i in range(width)]
    theirs = [one + shift + r * other_stride + i for r in range(n) for i in range(width)]
    got = ops._partly_the_same(one, stride, one + shift, other_stride, n, width)
    if mine == theirs or not set(mine) & set(theirs):
        assert not got or (stride != other_stride and max(mine[0], theirs[0]) <= min(mine[-1], theirs[-1]))
    else:
        assert got


@pytest.mark.gpu
def test_outputs_in_the_buffer_of_the_logits():
    n, V = 4, 1000
    edits = ops.LogitEdits(bias=ops.TokenBiases.from_rows([{3: 1.0}] * n, "cuda:0"))
    wide = torch.randn(n, 2 * V + 8, device="cuda:0")
    logits, beside = wide[:, :V], wide[:, V:2 * V]
    want = logits.clone()
    want[:, 3] += 1.0
    for out in (wide[:, 4:4 + V], wide[:, V - 1:2 * V - 1], torch.as_strided(wide, (n, V), (V + 1, 1))):
        with pytest.raises(ops.KernelError, match="overlaps"):
            ops.edit_logits(logits, edits, out)
    with pytest.raises(ops.KernelError, match="overlaps"):
        ops.edit_logits(logits[:-1], ops.LogitEdits(), logits[1:])
    assert torch.equal(ops.edit_logits(logits, edits, beside), want) and torch.equal(beside, want)
    assert torch.equal(ops.edit_logits(logits, edits, logits), want) and torch.equal(logits, want)
