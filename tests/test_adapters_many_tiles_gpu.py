"""More tiles of 16 rows than one launch of their kernel takes."""

import pytest
import torch

from reflex_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_million_rows_by_sixteens():
    R, K, N, rank = 16 * ops.ADAPTER_STEP_TILES + 5, 64, 24, 16
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(R, K, generator=g, device=DEV).to(torch.bfloat16)
    a = (torch.randn(2, 1, rank, K, generator=g, device=DEV) / 8).to(torch.bfloat16)
    b = torch.randn(2, N, rank, generator=g, device=DEV).to(torch.bfloat16)
    base = torch.randn(R, N, generator=g, device=DEV)
    scale = torch.tensor([0.5, 2.0], device=DEV)
    ids = torch.randint(-1, 2, (R,), generator=g, device=DEV, dtype=torch.int32)
    rows = ops.adapter_rows(ids, 2, 16)
    assert rows.n_tiles > ops.ADAPTER_STEP_TILES
    got = ops.adapter_add(base, x, ops.AdapterBank(a, b, scale, (N,)), rows)
    for i in (-1, 0, 1):
        some = (ids == i).nonzero()[-2000:, 0]  # the last ones: behind the launch's reach
        want, size = base[some].double(), base[some].double().abs()
        if i >= 0:
            low, low_size = x[some].double() @ a[i, 0].double().T, x[some].double().abs() @ a[i, 0].double().abs().T
            want = want + scale[i].double() * (low @ b[i].double().T)
            size = size + scale[i].double() * (low_size @ b[i].double().abs().T)
        # a step of 2^-24 for each product, sum and piece
        assert bool(((got[some].double() - want).abs() <= (K + 8 + rank + 4) * 2.0 ** -24 * size).all())
    ops.check_device_errors(DEV)
