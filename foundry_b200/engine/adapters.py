"""The adapters of an engine: names, places in the parts' banks, and the files they come from.

Every site (parts/adapters.py) has the same places; an adapter takes one of them everywhere. Loading one
writes its place on the current stream, where the engine's steps follow; a sequence holds its adapter's
place while it is open, and a place that is held is neither given away nor written.
"""
from __future__ import annotations

import json
import os
from typing import Dict, List, Mapping, Optional, Tuple

import torch

from ..kernels import ops
from ..parts.adapters import sites_of
from ..weights.safetensors_io import WeightFiles, parse_header


class AdapterError(ValueError):
    """An adapter that does not fit the model, or a name that is taken, unknown or in use."""


def read_folder(folder: str) -> Tuple[Dict[str, torch.Tensor], float]:
    """The tensors of adapter_model.safetensors and lora_alpha / r of adapter_config.json."""
    with open(os.path.join(folder, "adapter_config.json")) as handle:
        config = json.load(handle)
    for key in ("use_dora", "fan_in_fan_out", "lora_bias"):
        if config.get(key):
            raise AdapterError(f"{folder}: {key} is not supported")
    for key in ("rank_pattern", "alpha_pattern"):
        if config.get(key):
            raise AdapterError(f"{folder}: {key} is not supported")
    if config.get("bias", "none") != "none":
        raise AdapterError(f"{folder}: biases are not supported")
    try:
        rank, alpha = float(config["r"]), float(config["lora_alpha"])
    except (KeyError, TypeError, ValueError):
        raise AdapterError(f"{folder}: adapter_config.json needs r and lora_alpha") from None
    if rank <= 0:
        raise AdapterError(f"{folder}: r is {rank}")
    entries, _ = parse_header(os.path.join(folder, "adapter_model.safetensors"))
    files = WeightFiles(entries)
    scale = alpha / (rank ** 0.5 if config.get("use_rslora") else rank)
    return {name: files.tensor(name) for name in entries}, scale


def pairs_of(tensors: Mapping[str, torch.Tensor]) -> Dict[str, Tuple[torch.Tensor, torch.Tensor]]:
    """{projection: (A, B)} of tensors named `<projection>.lora_A.weight` and `.lora_B.weight`, with or
    without `base_model.model.` in front and an adapter's name before `weight`."""
    halves: Dict[str, Dict[str, torch.Tensor]] = {}
    for name, tensor in tensors.items():
        short = name[len("base_model.model."):] if name.startswith("base_model.model.") else name
        for half in ("lora_A", "lora_B"):
            at = short.find(f".{half}.")
            if at >= 0 and short.endswith("weight"):
                of = halves.setdefault(short[:at], {})
                if half in of:
                    raise AdapterError(f"{short[:at]}: {half} is given twice")
                of[half] = tensor
                break
        else:
            raise AdapterError(f"{name} is neither the A nor the B of a projection")
    lonely = sorted(p for p, h in halves.items() if len(h) != 2)
    if lonely:
        raise AdapterError(f"projections with only one of A and B: {lonely}")
    return {p: (h["lora_A"], h["lora_B"]) for p, h in halves.items()}


class AdapterStore:
    def __init__(self, model, max_adapters: int, max_rank: int, dtype: torch.dtype, device):
        if max_adapters < 1 or max_rank < 1:
            raise AdapterError(f"room for {max_adapters} adapters of rank {max_rank}")
        self.max_rank = (max_rank + 7) // 8 * 8  # the kernels' ranks
        self.dtype = dtype
        self.sites = sites_of(model.parts())
        if not self.sites:
            raise AdapterError(f"no part of {model.spec.architecture} takes adapters")
        # (the projections of one matrix stand side by side in its bank's ranks)
        most = ops.MAX_ADAPTER_RANK // max(len(site.names) for site in self.sites) // 8 * 8
        if self.max_rank > most:
            raise AdapterError(f"adapters of rank {max_rank}: up to {most} beside this model's projections")
        try:
            for site in self.sites:
                site.make(max_adapters, self.max_rank, dtype, device)
        except BaseException:
            for site in self.sites:  # (what was made before would hold its memory)
                site.bank = None
            raise
        self.places: Dict[str, int] = {}
        self._free: List[int] = list(range(max_adapters))
        self._held: Dict[int, int] = {}

    def place_of(self, name: str) -> int:
        try:
            return self.places[name]
        except KeyError:
            raise AdapterError(f"no adapter named {name!r}; loaded: {sorted(self.places)}") from None

    def hold(self, place: int) -> None:
        self._held[place] = self._held.get(place, 0) + 1

    def release(self, place: int) -> None:
        self._held[place] -= 1
        if not self._held[place]:
            del self._held[place]

    def load(self, name: str, source, scale: Optional[float] = None) -> None:
        if name in self.places:
            raise AdapterError(f"an adapter named {name!r} is loaded; unload it first")
        if not self._free:
            raise AdapterError(f"all {len(self.places)} places are taken: {sorted(self.places)}")
        if isinstance(source, (str, os.PathLike)):
            tensors, of_folder = read_folder(os.fspath(source))
            scale = of_folder if scale is None else scale
        else:
            tensors, scale = source, 1.0 if scale is None else scale
        scale = float(scale)
        if not abs(scale) <= torch.finfo(torch.float32).max:  # (what the banks hold it in)
            raise AdapterError(f"an adapter's scale is {scale}")
        pairs = pairs_of(tensors)
        self._check(name, pairs)
        place = self._free[0]  # taken when all of it is written: every site's numbers there are then this adapter's
        for site in self.sites:
            site.write(place, pairs, scale)
        self._free.pop(0)
        self.places[name] = place

    def _check(self, name: str, pairs) -> None:
        known = {p: (rows, site.in_features) for site in self.sites for p, rows in site.names}
        wrong = []
        for p, (a, b) in sorted(pairs.items()):
            if p not in known:
                wrong.append(f"{p}: not a projection that takes adapters")
                continue
            rows, cols = known[p]
            if a.dim() != 2 or b.dim() != 2 or a.shape[1] != cols or b.shape[0] != rows or \
                    a.shape[0] != b.shape[1]:
                wrong.append(f"{p}: A {tuple(a.shape)}, B {tuple(b.shape)} beside [{rows}, {cols}]")
            elif a.shape[0] > self.max_rank:
                wrong.append(f"{p}: rank {a.shape[0]}, room for {self.max_rank}")
            elif not all(torch.isfinite(t.to(self.dtype)).all() for t in (a, b)):
                wrong.append(f"{p}: not finite (as {self.dtype})")
        if not pairs:
            wrong.append("no tensors")
        if wrong:
            raise AdapterError(f"adapter {name!r} does not fit: " + "; ".join(wrong))

    def unload(self, name: str) -> None:
        place = self.place_of(name)
        if place in self._held:
            raise AdapterError(f"adapter {name!r} is in use by {self._held[place]} open sequences")
        del self.places[name]
        for site in self.sites:
            site.clear(place)
        self._free.append(place)
