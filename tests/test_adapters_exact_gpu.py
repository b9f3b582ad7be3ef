"""Adapters beside a projection where exact arithmetic leaves little of large low-rank rows: what a product hands to the
other keeps 24 bits."""

import pytest
import torch

from reflex_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)]


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("rows,tile", [(1, 16), (9, 16), (300, 16), (1, 128), (130, 128), (600, 128)])
@pytest.mark.parametrize("cols,rank,woven", [((128,), 16, False), ((64, 64, 64), 64, False), ((96,), 128, False),
                                             ((64, 64), 32, True), ((64, 64), 64, True)])
def test_low_rank_rows_keep_24_bits(rows, tile, cols, rank, woven, dtype, out):
    """A x has 1 + 2^-9 + 2^-18 and 1 + 2^-9, which 24 bits hold; B takes their difference, 2^-18, exactly."""
    K = 256
    x = torch.zeros(rows, K, device=DEV, dtype=dtype)
    x[:, 0], x[:, 100], x[:, 255] = 1.0, 2.0 ** -9, 2.0 ** -18
    a = torch.zeros(1, len(cols), rank, K, device=DEV, dtype=dtype)
    a[:, :, 0], a[:, :, rank - 1, :255] = 1.0, 1.0
    b = torch.zeros(1, sum(cols), rank, device=DEV, dtype=dtype)
    b[:, :, 0], b[:, :, rank - 1] = 1.0, -1.0
    bank = ops.AdapterBank(a, b, torch.ones(1, device=DEV), cols, woven=woven)
    ids = torch.zeros(rows, dtype=torch.int32, device=DEV)
    base = torch.zeros(rows, sum(cols), device=DEV, dtype=out)
    got = ops.adapter_add(base, x, bank, ops.adapter_rows(ids, 1, tile))
    assert bool((got == 2.0 ** -18).all()), got.unique().tolist()[:4]
    ops.check_device_errors(DEV)
