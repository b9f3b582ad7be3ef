"""A token a row where a row's CTAs have next to nothing to load: launches one behind the other, in which a CTA is soon
done with its own piece and writes to the others'."""

import numpy as np
import pytest
import torch

from reflex_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("B,V", [(1, 65537), (4, 70001), (5, 33000), (40, 16385), (200, 8193)])
def test_short_pieces_in_launches_one_behind_the_other(B, V):
    rng = np.random.default_rng(B)
    l = torch.tensor(rng.normal(0, 1, (B, V)).astype(np.float32), device=DEV)
    at = torch.tensor(rng.permutation(V)[:B], device=DEV)
    l[torch.arange(B), at] = 50.0  # the rest of the row is e^-45 of it or less
    T, u = torch.full((B,), 0.9, device=DEV), torch.full((B,), 0.5, device=DEV)
    p, cold = torch.full((B,), 0.9, device=DEV), torch.zeros(B, device=DEV)
    outs = [torch.full((B,), -1, dtype=torch.int32, device=DEV) for _ in range(300)]
    for i, out in enumerate(outs):
        ops.sample_rows(l, cold if i % 3 == 0 else T, u, top_p=p if i % 3 == 1 else None, out=out)
    for out in outs:
        assert torch.equal(out.long(), at)
