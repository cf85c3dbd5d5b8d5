"""The planes of a large bank's adapters are made for as many tokens at a time as their room takes."""
import pytest
import torch

from foundry_b200.kernels import ops

DEV = "cuda:0"


@pytest.mark.parametrize("T", [300, 8192])
@pytest.mark.parametrize("slots", [1, 8, 64, 256, 1024])
@pytest.mark.parametrize("rank", [8, 64, 200, 512])
def test_the_room_of_the_planes(T, slots, rank):
    """256 MB, or what one block of 256 tokens takes (every place's plane: 134 MB at the most)."""
    tokens = ops._planes_piece(T, slots, rank)
    most = min(slots, 256, T)
    size = lambda n: -(-n // 256) * most * 256 * ops._plane_width(rank) * 2  # noqa: E731
    assert 0 < tokens <= T and (tokens == T or tokens % 256 == 0)
    assert size(tokens) <= 1 << 28
    assert tokens == T or size(tokens + 256) > 1 << 28  # no more pieces than it takes


@pytest.mark.gpu
@pytest.mark.parametrize("T", [300, 512, 769, 2000])
def test_pieces_are_the_whole(T, monkeypatch):
    g = torch.Generator(device=DEV).manual_seed(T)
    make = lambda *shape: torch.randn(*shape, generator=g, device=DEV).bfloat16()  # noqa: E731
    K, N, R, S = 256, 400, 24, 5
    x, w = make(T, K + 8)[:, :K], make(N, K) * 0.05
    bank = ops.AdapterBank(make(S, R, K) / 16, make(S, N, R), torch.rand(S, generator=g, device=DEV))
    index = torch.randint(-1, S, (T,), generator=g, device=DEV, dtype=torch.int32)
    monkeypatch.setattr(ops, "_planes_pay", lambda *sizes: True)
    want = ops.adapted_product(x, w, bank, index)
    sizes = []
    made = ops._adapted_planes
    monkeypatch.setattr(ops, "_adapted_planes", lambda x, *more: sizes.append(x.shape[0]) or made(x, *more))
    for room in (1, 2 * 5 * 256 * 64 * 2):  # a block at a time, and two
        monkeypatch.setattr(ops, "PLANES_ROOM", room)
        sizes.clear()
        assert torch.equal(ops.adapted_product(x, w, bank, index), want)
        assert len(sizes) == -(-T // (256 if room == 1 else 512))


@pytest.mark.gpu
def test_a_long_prompt_beside_a_large_bank_takes_little_memory():
    T, K, N, R, S = 8192, 256, 512, 256, 256
    x = torch.randn(T, K, device=DEV).bfloat16()
    w = torch.zeros(N, K, dtype=torch.bfloat16, device=DEV)
    bank = ops.AdapterBank(torch.zeros(S, R, K, dtype=torch.bfloat16, device=DEV), torch.zeros(S, N, R, dtype=torch.bfloat16, device=DEV),
                           torch.ones(S, device=DEV))
    index = torch.full((T,), 3, dtype=torch.int32, device=DEV)
    assert ops._planes_pay(T, N, S, R)
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.adapted_product(x, w, bank, index)
    assert torch.cuda.max_memory_allocated() - before < (1 << 28) + (1 << 26)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_long_prompts_gated_pairs_take_a_pieces_room(dtype, act):
    """32-bit gate and up rows stand in memory for 8,192 tokens at a time."""
    T, K, I, R = 20000, 64, 512, 8
    g = torch.Generator(device=DEV).manual_seed(0)
    make = lambda *shape: torch.randn(*shape, generator=g, device=DEV).to(dtype)  # noqa: E731
    x, w = make(T, K), make(2 * I, K) * 0.1
    bank = ops.AdapterBank(make(3, R, K) / 8, make(3, 2 * I, R) * 0.1, torch.ones(3, device=DEV))
    index = torch.arange(T, device=DEV, dtype=torch.int32) * 5 // T % 4
    out = torch.empty(T, I, dtype=dtype, device=DEV)
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.adapted_silu_mul(x, w, bank, index, out, act=act)
    assert torch.cuda.max_memory_allocated() - before < 2.5 * 8192 * 2 * I * 4
    for t in (0, 8191, 8192, 16383, 16384, T - 1):
        some = torch.empty(1, I, dtype=dtype, device=DEV)
        ops.adapted_silu_mul(x[t:t + 1], w, bank, index[t:t + 1], some, act=act)
        assert torch.allclose(out[t].float(), some[0].float(), rtol=2.0 ** -6, atol=1e-4)
