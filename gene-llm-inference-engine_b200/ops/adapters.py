"""Low-rank adapters of a projection, several kept side by side, and the step's rows that use them.

An adapter of a projection y = W x is a pair of matrices, y += scale * up (down x) with ``down`` [rank, in] and ``up``
[out, rank]. ``AdapterSet`` holds the pairs of one projection for a fixed number of slots on the device, stacked as
``kernels.adapter_product`` reads them; ranks below the set's are filled up with zeros. A projection that stacks several
([q; k; v], [gate; up]) has a pair per part. ``AdapterStep`` is what all adapted projections of an engine share: the plan of the rows of the
step that is being run (None: no row of it has an adapter, and nothing of this runs).
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import kernels


class AdapterStep:
    """The rows of the current step in the adapters' order, for every adapted projection."""

    def __init__(self, slots: int, max_rows: int, device: torch.device):
        self.slots = slots
        self.plan: Optional[kernels.AdapterPlan] = None
        self._buffer = torch.empty(max(1, kernels.adapter_plan_size(max_rows, slots)), dtype=torch.int32, device=device)

    def begin(self, row_adapter: Optional[torch.Tensor], used: Optional[int] = None) -> None:
        """``row_adapter`` [rows] int32 on the device: every row's slot, or a negative number; None: no adapters in this step.
        ``used``: so many different ones at most."""
        self.plan = None if row_adapter is None else kernels.adapter_plan(row_adapter, self.slots, self._buffer, min(self.slots, used or self.slots))


class AdapterSet:
    def __init__(self, slots: int, rank: int, in_features: int, widths: Sequence[int], dtype: torch.dtype, device: torch.device):
        """``widths``: the output columns of the parts stacked in the projection."""
        self.check_sizes(slots, rank, widths)
        self.slots, self.rank = slots, self.rank_held(rank)
        self.widths = [int(n) for n in widths]
        self.in_features, self.out_features = in_features, sum(self.widths)
        self.down = torch.zeros(slots, len(self.widths) * self.rank, in_features, dtype=dtype, device=device)
        self.up = torch.zeros(slots, self.out_features, self.rank, dtype=dtype, device=device)
        self.scales = torch.zeros(slots, dtype=torch.float32, device=device)

    @staticmethod
    def rank_held(rank: int) -> int:
        return (rank + 3) // 4 * 4                                  # (pieces of four ranks are read at once)

    @classmethod
    def check_sizes(cls, slots: int, rank: int, widths: Sequence[int]) -> None:
        """Raises ``ValueError`` for sizes that the products do not take."""
        if slots < 1 or rank < 1 or not widths:
            raise ValueError("adapters: slots, rank and parts must be positive")
        if slots > kernels.ADAPTER_ADAPTERS_MOST:
            raise ValueError(f"adapters: {slots} slots (at most {kernels.ADAPTER_ADAPTERS_MOST})")
        if len(widths) * cls.rank_held(rank) > kernels.ADAPTER_RANKS_MOST:
            raise ValueError(f"adapters: rank {rank} in a projection that stacks {len(widths)} (at most {kernels.ADAPTER_RANKS_MOST // len(widths) // 4 * 4})")

    def clear(self, slot: int) -> None:
        """The slot's adapter is none: its rows get zeros added."""
        self._check(slot)
        self.down[slot].zero_()
        self.up[slot].zero_()
        self.scales[slot] = 0.0

    def check(self, slot: int, pairs: Sequence) -> None:
        """Raises ``ValueError`` where ``put`` cannot take the pairs."""
        self._check(slot)
        if len(pairs) != len(self.widths):
            raise ValueError(f"adapters: {len(pairs)} pairs for {len(self.widths)} parts")
        for i, pair in enumerate(pairs):
            if pair is None:
                continue
            down, up = pair
            if down.dim() != 2 or up.dim() != 2 or down.shape[1] != self.in_features or up.shape[0] != self.widths[i] or down.shape[0] != up.shape[1]:
                raise ValueError(f"adapters: down {tuple(down.shape)} and up {tuple(up.shape)} do not fit a part of "
                                 f"{self.in_features} inputs and {self.widths[i]} outputs")
            if down.shape[0] > self.rank:
                raise ValueError(f"adapters: rank {down.shape[0]} exceeds {self.rank}")

    def put(self, slot: int, pairs: Sequence, scale: float) -> None:
        """``pairs``: a (down, up) for every part, or None for a part without one."""
        self.check(slot, pairs)
        self.clear(slot)
        at = 0
        for i, (pair, n) in enumerate(zip(pairs, self.widths)):
            if pair is not None:
                down, up = pair
                r = down.shape[0]
                self.down[slot, i * self.rank:i * self.rank + r] = down.to(self.down)
                self.up[slot, at:at + n, :r] = up.to(self.up)
            at += n
        self.scales[slot] = float(scale)

    def add(self, x: torch.Tensor, plan: kernels.AdapterPlan, out: torch.Tensor) -> None:
        """out[t] += the adapter of row t on x[t]."""
        kernels.adapter_product(x, self.down, self.up, self.scales, plan, out, self.widths)

    def _check(self, slot: int) -> None:
        if not 0 <= slot < self.slots:
            raise ValueError(f"adapters: slot {slot} is outside 0..{self.slots - 1}")
