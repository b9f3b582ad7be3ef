"""The adapters of a part's projections, side by side on the device.

A part whose projections may have adapters says `takes_adapters` and offers `adapter_banks(pairs, scales)`: `pairs`
maps a role of its `tensor_specs` to the adapters' (A, B) for that matrix, one a loaded adapter (None where an adapter
leaves it as it is).  What it returns is put into its `adapters`.  In a step with adapters (`ops.active_adapters()`) it
adds them to what the shared product gave.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from .. import ops


def make_bank(pairs: Sequence[Sequence], cols: Sequence[int], width: int, scales: Sequence[float], dtype: torch.dtype,
              device, woven: bool = False) -> Optional[ops.AdapterBank]:
    """`pairs[s][i]`: adapter i's (A [r, width], B [cols[s], r]) for part s of a stacked projection, or None; None
    comes back where no adapter changes the projection."""
    ranks = [max((p[i][0].shape[0] for p in pairs if p[i] is not None), default=0) for i in range(len(scales))]
    rank, N = max(ranks, default=0), sum(cols)
    if rank == 0:
        return None
    a = torch.zeros((len(scales), len(cols), rank, width), dtype=dtype)
    b = torch.zeros((len(scales), N, rank), dtype=dtype)
    for s, part in enumerate(pairs):
        first = sum(cols[:s])
        for i, pair in enumerate(part):
            if pair is not None:
                r = pair[0].shape[0]
                a[i, s, :r] = pair[0].to(dtype)
                (b[i, s::2] if woven else b[i, first:first + cols[s]])[:, :r] = pair[1].to(dtype)
    return ops.AdapterBank(a.to(device), b.to(device), torch.tensor(scales, dtype=torch.float32, device=device), cols,
                           woven=woven, ranks=torch.tensor(ranks, dtype=torch.int32, device=device))


def add(y: torch.Tensor, x: torch.Tensor, bank: Optional[ops.AdapterBank]) -> torch.Tensor:
    """What the step's adapters add to `y`, the shared product of `x`, in place."""
    rows = ops.active_adapters()
    return y if bank is None or rows is None else ops.adapter_add(y, x, bank, rows, out=y)
