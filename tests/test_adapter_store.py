"""The adapters of an engine on the host: names, places, what fits and what is refused."""
import types

import pytest
import torch

from foundry_b200.engine.adapters import AdapterError, AdapterStore, pairs_of
from foundry_b200.parts.adapters import AdapterSite


def store(places=2, rank=8, dtype=torch.float32):
    part = types.SimpleNamespace()
    order = torch.tensor([1, 0, 3, 2, 5, 4, 6])
    part.sites = [AdapterSite([("a.q", 4), ("a.k", 2), ("a.v", 1)], 6, order), AdapterSite([("a.o", 6)], 4)]
    part.adapter_sites = lambda: part.sites
    model = types.SimpleNamespace(parts=lambda: [part, types.SimpleNamespace()], spec=types.SimpleNamespace(architecture="Toy"))
    return AdapterStore(model, places, rank, dtype, "cpu"), part.sites


def pair(name, rows, cols, r=3, seed=0):
    g = torch.Generator().manual_seed(seed)
    return {f"{name}.lora_A.weight": torch.randn(r, cols, generator=g), f"{name}.lora_B.weight": torch.randn(rows, r, generator=g)}


def test_a_bank_holds_its_projections_side_by_side_in_the_matrixs_order():
    held, sites = store()
    given = {**pair("a.q", 4, 6), **pair("a.v", 1, 6, r=8, seed=1)}
    held.load("x", given, 0.5)
    bank, x = sites[0].bank, torch.randn(5, 6)
    assert bank.a.shape == (2, 24, 6) and bank.b.shape == (2, 7, 24) and float(bank.scales[0]) == 0.5
    wide = torch.zeros(5, 7)
    wide[:, :4] = x @ given["a.q.lora_A.weight"].T @ given["a.q.lora_B.weight"].T
    wide[:, 6:] = x @ given["a.v.lora_A.weight"].T @ given["a.v.lora_B.weight"].T
    assert torch.allclose(x @ bank.a[0].T @ bank.b[0].T, wide[:, sites[0].order], atol=1e-5)
    assert not sites[1].bank.a.any() and not bank.a[1].any()


def test_places_are_given_back_and_never_while_they_are_held():
    held, sites = store()
    held.load("x", pair("a.o", 6, 4))
    held.load("y", pair("a.o", 6, 4, seed=1))
    held.hold(held.place_of("x"))
    for refused in (lambda: held.load("z", pair("a.o", 6, 4)), lambda: held.load("x", pair("a.o", 6, 4)),
                    lambda: held.unload("x"), lambda: held.unload("w"), lambda: held.place_of("w")):
        with pytest.raises(AdapterError):
            refused()
    held.release(held.place_of("x"))
    held.unload("x")
    assert not sites[1].bank.a[0].any() and not sites[1].bank.b[0].any()
    held.load("z", pair("a.o", 6, 4, seed=2))
    assert held.place_of("z") == 0


@pytest.mark.parametrize("tensors,what", [
    ({}, "no tensors"), (pair("a.p", 4, 6), "not a projection"), (pair("a.o", 6, 5), "beside"),
    (pair("a.o", 6, 4, r=9), "rank 9"), ({"a.o.lora_A.weight": torch.zeros(1, 4)}, "only one"),
    ({"a.o.weight": torch.zeros(1, 4)}, "neither")])
def test_what_does_not_fit_is_refused(tensors, what):
    with pytest.raises(AdapterError, match=what):
        store()[0].load("x", tensors)
    with pytest.raises(AdapterError, match="scale"):
        store()[0].load("x", pair("a.o", 6, 4), float("inf"))


@pytest.mark.parametrize("half", ["lora_A", "lora_B"])
@pytest.mark.parametrize("value,dtype,fits", [(float("nan"), torch.float32, False), (float("inf"), torch.float32, False),
                                              (3.4e38, torch.float32, True), (3.4e38, torch.bfloat16, False),
                                              (3.3e38, torch.bfloat16, True), (1e300, torch.float32, False)])
def test_numbers_are_finite_in_the_type_that_holds_them(half, value, dtype, fits):
    given = {n: t.double() for n, t in pair("a.o", 6, 4).items()}
    given[f"a.o.{half}.weight"][1, 1] = value
    if fits:
        store(dtype=dtype)[0].load("x", given)
        return
    with pytest.raises(AdapterError, match="not finite"):
        store(dtype=dtype)[0].load("x", given)


def test_a_projection_that_is_given_twice_is_refused():
    given = pair("a.o", 6, 4)
    again = {f"base_model.model.{n}": t for n, t in given.items()}
    assert set(pairs_of(again)) == {"a.o"}
    with pytest.raises(AdapterError, match="twice"):
        pairs_of({**given, **again})
    with pytest.raises(AdapterError, match="twice"):
        pairs_of({**given, "a.o.lora_B.other.weight": given["a.o.lora_B.weight"]})
