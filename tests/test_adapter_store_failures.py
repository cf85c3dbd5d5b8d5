"""What an engine's adapters do where a step of theirs fails, on the host."""
import types

import pytest
import torch

from foundry_b200.engine.adapters import AdapterError, AdapterStore
from foundry_b200.kernels import ops
from foundry_b200.parts.adapters import AdapterSite


def model_of(sites):
    part = types.SimpleNamespace(adapter_sites=lambda: sites)
    return types.SimpleNamespace(parts=lambda: [part], spec=types.SimpleNamespace(architecture="Toy"))


def sites():
    return [AdapterSite([("a.o", 6)], 8), AdapterSite([("a.q", 4), ("a.k", 2), ("a.v", 1)], 8), AdapterSite([("a.g", 3), ("a.u", 3)], 8)]


def pairs(rank=2):
    return {f"{name}.lora_{half}.weight": torch.ones(shape) for name, rows in (("a.o", 6), ("a.q", 4))
            for half, shape in (("A", (rank, 8)), ("B", (rows, rank)))}


@pytest.mark.parametrize("rank", [161, 168, 169, 512])
def test_the_largest_rank_is_that_of_the_fused_matrices(rank):
    """Three projections of one matrix share its bank's ranks (ops.MAX_ADAPTER_RANK)."""
    some = sites()
    if rank <= ops.MAX_ADAPTER_RANK // 3 // 8 * 8:
        assert AdapterStore(model_of(some), 2, rank, torch.float32, "cpu").max_rank == 168
        return
    with pytest.raises(AdapterError, match=f"rank {rank}: up to 168 beside this model"):
        AdapterStore(model_of(some), 2, rank, torch.float32, "cpu")
    assert all(s.bank is None for s in some)  # nothing was made
    assert AdapterStore(model_of(some[:1]), 2, rank, torch.float32, "cpu").max_rank >= rank


def test_a_place_is_taken_by_what_is_written():
    """An adapter whose writing failed (no memory, say) leaves its place to the next one, and nothing of itself there."""
    some = sites()
    store = AdapterStore(model_of(some), 1, 8, torch.float32, "cpu")
    write = some[1].write

    def fails(*args):
        write(*args)
        raise MemoryError("no room")
    some[1].write = fails
    for _ in range(3):
        with pytest.raises(MemoryError):
            store.load("x", pairs())
    assert store.places == {}
    some[1].write = write
    store.load("y", {k: v for k, v in pairs().items() if k.startswith("a.q")}, 2.0)
    assert store.place_of("y") == 0 and not some[0].bank.b.any() and not some[0].bank.a.any()


def test_room_that_cannot_be_made_leaves_none():
    some = sites()
    some[2].make = lambda *args: (_ for _ in ()).throw(MemoryError("no room"))
    with pytest.raises(MemoryError):
        AdapterStore(model_of(some), 1, 8, torch.float32, "cpu")
    assert all(s.bank is None for s in some)


@pytest.mark.parametrize("scale", [1e39, -1e39, float("inf"), float("nan")])
def test_a_scale_is_finite_in_the_type_that_holds_it(scale):
    some = sites()
    store = AdapterStore(model_of(some), 1, 8, torch.float32, "cpu")
    with pytest.raises(AdapterError, match="scale"):
        store.load("x", pairs(), scale)
    store.load("x", pairs(), 3e38)
    assert torch.isfinite(some[0].bank.scales).all()
