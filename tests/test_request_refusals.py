"""What the operators of single requests refuse, before anything runs: on tensors of the CPU, and (the
checks that come first) on tensors without memory."""
import pytest
import torch

from foundry_b200.kernels import ops


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_a_history_and_its_bits_have_one_size():
    ops.TokenHistory(i32(3, 65), i32(3, 3))
    for counts, seen in ((i32(3, 65), i32(3, 2)), (i32(3, 65), i32(2, 3)), (i32(65), i32(3))):
        with pytest.raises(ops.KernelError, match="history"):
            ops.TokenHistory(counts, seen)


def test_biases_are_three_lists():
    with pytest.raises(ops.KernelError, match="biases"):
        ops.TokenBiases(i32(3), i32(5), torch.zeros(4))
    b = ops.TokenBiases.from_rows([{9: 1.0, 2: -3.5}, None, {0: 4.0}], "cpu")
    assert b.starts.tolist() == [0, 2, 2, 3] and b.ids.tolist() == [2, 9, 0]
    assert b.values.tolist() == [-3.5, 1.0, 4.0]


def test_edits_come_in_pairs():
    history = ops.TokenHistory(i32(2, 40), i32(2, 2))
    for given in (dict(history=history), dict(history_rows=i32(1)), dict(repetition=torch.ones(1)),
                  dict(allowed=i32(1, 2)), dict(allowed_rows=i32(1))):
        with pytest.raises(ops.KernelError):
            ops.LogitEdits(**given)


def test_edits_fit_the_rows():
    cpu = -1  # the number of the CPU's tensors
    history = ops.TokenHistory(i32(2, 40), i32(2, 2))
    fits = ops.LogitEdits(history, i32(3), torch.ones(3), allowed=i32(1, 2), allowed_rows=i32(3))
    fits.packed(3, 40, cpu)
    for n, vocab in ((2, 40), (3, 41), (3, 64)):
        with pytest.raises(ops.KernelError):
            fits.packed(n, vocab, cpu)
    bad = [ops.LogitEdits(history, torch.zeros(3, dtype=torch.int64)),
           ops.LogitEdits(history, i32(6)[::2]),
           ops.LogitEdits(history, i32(3), presence=torch.ones(3, dtype=torch.float64)),
           ops.LogitEdits(history, i32(3), frequency=torch.ones(2)),
           ops.LogitEdits(allowed=i32(1, 3), allowed_rows=i32(3)),
           ops.LogitEdits(bias=ops.TokenBiases(i32(3), i32(4), torch.zeros(4))),
           ops.LogitEdits(bias=ops.TokenBiases(i32(4), i32(4), torch.zeros(4, dtype=torch.float64)))]
    for edits in bad:
        with pytest.raises(ops.KernelError):
            edits.packed(3, 40, cpu)


def test_logits_are_float32_rows_on_the_device():
    for logits in (torch.zeros(2, 40), torch.zeros(2, 40, dtype=torch.bfloat16), torch.zeros(40)):
        with pytest.raises(ops.KernelError):
            ops.edit_logits(logits, ops.LogitEdits())
        with pytest.raises(ops.KernelError):
            ops.sample_tokens(logits, ops.SampleRules())
    with pytest.raises(ops.KernelError, match="known"):
        ops.record_tokens(ops.TokenHistory(i32(2, 40), i32(2, 2)), i32(1), i32(1), "forgotten")
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.record_tokens(ops.TokenHistory(i32(2, 40), i32(2, 2)), i32(1), i32(1))


def test_adapters_of_one_bank():
    a, b, scales = torch.zeros(2, 16, 64), torch.zeros(2, 32, 16), torch.ones(2)
    bank = ops.AdapterBank(a, b, scales)
    assert (bank.slots, bank.rank) == (2, 16)
    for other in ((a[0], b, scales), (a, b[:1], scales), (a, b[:, :, :8], scales), (a, b, scales[:1]),
                  (a[:0], b[:0], scales[:0]), (a[:, :12], b[:, :, :12], scales),
                  (torch.zeros(2, 520, 64), torch.zeros(2, 32, 520), scales)):
        with pytest.raises(ops.KernelError, match="adapters"):
            ops.AdapterBank(*other)


def test_an_adapted_product_of_foreign_sizes():
    bank = ops.AdapterBank(torch.zeros(2, 16, 64), torch.zeros(2, 32, 16), torch.ones(2))
    x, w = torch.zeros(3, 64), torch.zeros(32, 64)
    for other in ((x[:, :56], w), (x, w[:16]), (x, w.bfloat16()), (x[0], w), (torch.zeros(3, 72), torch.zeros(32, 72))):
        with pytest.raises(ops.KernelError):
            ops.adapted_product(*other, bank, i32(3))
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.adapted_product(x, w, bank, i32(3))
