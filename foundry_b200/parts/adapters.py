"""Room for low-rank adapters beside a projection.

A site is one matrix of a part, which may hold several named projections (q, k and v; gate and up). An
adapter gives some of them A [r, in] and B [out, r], y += scale (x A^T) B^T, and here they are one bank of
the matrix (`ops.AdapterBank`): the projections' A one below the other, their B in the rows that the matrix
has for them (whatever their order is: rotation partners side by side, gate and up interleaved) and in the
columns of their own ranks, zeros elsewhere.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch

from ..kernels import ops


class AdapterSite:
    def __init__(self, names: Sequence[Tuple[str, int]], in_features: int,
                 order: Optional[torch.Tensor] = None):
        self.names = list(names)  # (projection's full name, rows)
        self.in_features = in_features
        self.order = order        # row p of the matrix is row order[p] of the projections one below the other
        self.bank: Optional[ops.AdapterBank] = None
        self.rank = 0             # of one projection

    @property
    def out_features(self) -> int:
        return sum(rows for _, rows in self.names)

    def make(self, places: int, rank: int, dtype: torch.dtype, device) -> None:
        self.rank = rank
        total = rank * len(self.names)
        self.bank = ops.AdapterBank(
            torch.zeros(places, total, self.in_features, dtype=dtype, device=device),
            torch.zeros(places, self.out_features, total, dtype=dtype, device=device),
            torch.zeros(places, dtype=torch.float32, device=device))

    def clear(self, place: int) -> None:
        self.bank.a[place].zero_()
        self.bank.b[place].zero_()
        self.bank.scales[place] = 0.0

    def write(self, place: int, given: Dict[str, Tuple[torch.Tensor, torch.Tensor]],
              scale: float) -> None:
        """The adapter's A and B of this site's projections (none of one: zeros)."""
        bank = self.bank
        a = torch.zeros_like(bank.a[place])
        b = torch.zeros_like(bank.b[place])
        row = 0
        for i, (name, rows) in enumerate(self.names):
            if name in given:
                low, up = (t.to(device=a.device, dtype=a.dtype) for t in given[name])
                r = low.shape[0]
                a[i * self.rank:i * self.rank + r] = low
                b[row:row + rows, i * self.rank:i * self.rank + r] = up
            row += rows
        bank.a[place] = a
        bank.b[place] = b if self.order is None else b.index_select(0, self.order.to(b.device))
        bank.scales[place] = float(scale)


def sites_of(parts) -> List[AdapterSite]:
    """The sites of the parts that take adapters."""
    found: List[AdapterSite] = []
    for part in parts:
        offer = getattr(part, "adapter_sites", None)
        if callable(offer):
            found += offer()
    return found
