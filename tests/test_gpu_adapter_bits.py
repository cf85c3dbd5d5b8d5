"""How many bits of a rank number reach the adapters' results, on each of the ways that they take. Whole numbers:
every product and sum of them is exact in 32 bits, so a result is right or it is not."""
import numpy as np
import pytest
import torch

import plain_requests as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from foundry_b200.kernels import ops
    return ops


@pytest.fixture(params=["by the rule", "behind the paired product's K", "behind K of a few rows"])
def way(request, ops, monkeypatch):
    """Where the rank numbers meet B: as the sizes' rules say, or one of the ways for all sizes that it takes."""
    if request.param == "behind the paired product's K":
        monkeypatch.setattr(ops, "_planes_pay", lambda T, N, slots, rank: T > 64 and N >= 128)
    elif request.param == "behind K of a few rows":
        monkeypatch.setattr(ops, "_rows_pay", lambda T, N, slots, rank: T <= 64)
    return ops


def whole_numbers(ops, T, K, N, R, S, seed=0):
    """|rank number| <= 16 K < 2^15 before a scale of a power of two, and nearly all of them past 2^8."""
    g = torch.Generator().manual_seed(seed + 1000 * T + K + N + R)
    pick = lambda most, *shape: torch.randint(-most, most + 1, shape, generator=g).bfloat16().to(DEV)  # noqa: E731
    x, w, a = pick(4, T, K), pick(2, N, K), pick(4, S, R, K)
    b = pick(1, S, N, R)
    scales = (2.0 ** torch.randint(-2, 3, (S,), generator=g)).to(DEV)
    index = torch.randint(-1, S, (T,), generator=g).to(torch.int32).to(DEV)
    return x, w, ops.AdapterBank(a, b, scales), index


def sums_of(x, w, bank, index):
    host = lambda t: t.float().cpu().numpy()  # noqa: E731
    return plain.adapted(*(host(t) for t in (x, w, bank.a, bank.b, bank.scales)), index.cpu().numpy())


@pytest.mark.parametrize("T", [1, 8, 16, 17, 40, 64, 65, 200, 300])
@pytest.mark.parametrize("K,N,R,S", [(512, 136, 8, 1), (1024, 200, 16, 4), (520, 264, 24, 3), (512, 128, 32, 9), (264, 136, 40, 20),
                                     (512, 400, 64, 3), (128, 256, 72, 5), (512, 136, 200, 2), (64, 128, 512, 3)])
def test_rank_numbers_of_sixteen_bits_arrive_whole(way, T, K, N, R, S):
    ops = way
    x, w, bank, index = whole_numbers(ops, T, K, N, R, S)
    want, _, much = sums_of(x, w, bank, index)
    assert much.max() < 1 << 22  # (every partial sum is a whole number of quarters: exact)
    got = ops.adapted_product(x, w, bank, index, out_dtype=torch.float32)
    assert np.array_equal(got.cpu().numpy(), want.astype(np.float32))


@pytest.mark.parametrize("T,K,N,R,S", [(64, 16392, 264, 64, 20), (40, 26216, 136, 64, 3), (300, 4096, 512, 64, 3)])
def test_rank_numbers_of_the_tensor_cores_arrive_whole(ops, T, K, N, R, S):
    """(The numbers and their sums take fewer bits where the matrix of x has a few ones a row.)"""
    assert ops._low_pays(T, K, S, R)
    x, w, bank, index = whole_numbers(ops, T, K, N, R, S)
    g = torch.Generator().manual_seed(T)
    x *= (torch.rand(T, K, generator=g) < 500 / K).to(DEV)
    want, _, much = sums_of(x, w, bank, index)
    assert much.max() < 1 << 22
    got = ops.adapted_product(x, w, bank, index, out_dtype=torch.float32)
    assert np.array_equal(got.cpu().numpy(), want.astype(np.float32))


@pytest.mark.parametrize("T", [9, 48, 70, 300])
@pytest.mark.parametrize("K,N,R,S", [(64, 256, 16, 4), (128, 520, 48, 3), (256, 648, 128, 5)])
def test_thirty_two_bit_results_are_within_the_halves_of_a_rank_number(way, T, K, N, R, S):
    """A rank number as the sum of two bfloat16 numbers: the second one's rounding, 2^-8 of at most 2^-8 of it."""
    ops = way
    g = torch.Generator().manual_seed(T + K)
    normal = lambda *shape: torch.randn(*shape, generator=g).bfloat16().to(DEV)  # noqa: E731
    bank = ops.AdapterBank(normal(S, R, K) / K ** 0.5, normal(S, N, R), (0.5 + torch.rand(S, generator=g)).to(DEV))
    x, w, index = normal(T, K), normal(N, K) * 0.05, torch.randint(-1, S, (T,), generator=g).to(torch.int32).to(DEV)
    want, size, much = sums_of(x, w, bank, index)
    got = ops.adapted_product(x, w, bank, index, out_dtype=torch.float32)
    bound = (K + 2 * R + 8) * 2.0 ** -24 * much + 2.0 ** -16 * size + 2.0 ** -24 * np.abs(want)
    off = np.abs(got.double().cpu().numpy() - want)
    assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("T", [12, 40, 100, 300])
def test_rank_numbers_past_the_largest_of_bfloat16(way, T):
    """A number between the largest of bfloat16 and of 32 bits rounds to infinity there; its second half is none then,
    and the results are infinite, as those of a 32-bit sum of as much would be."""
    ops = way
    x = torch.ones(T, 64, dtype=torch.bfloat16, device=DEV)
    a = torch.zeros(1, 8, 64, dtype=torch.bfloat16, device=DEV)
    a[0, 0, 0] = 2.0 ** 127
    a[0, 0, 1] = 2.0 ** 127 * (1 - 2.0 ** -8)
    a[0, 0, 2] = 2.0 ** 127 * 2.0 ** -9
    b = torch.zeros(1, 128, 8, dtype=torch.bfloat16, device=DEV)
    b[0, :, 0] = 4.0
    bank = ops.AdapterBank(a, b, torch.ones(1, device=DEV))
    index = torch.zeros(T, dtype=torch.int32, device=DEV)
    got = ops.adapted_product(x, torch.zeros(128, 64, dtype=torch.bfloat16, device=DEV), bank, index, out_dtype=torch.float32)
    assert (got == float("inf")).all()
