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


@pytest.mark.parametrize("rows,tile,K,chain", [(16, 16, 12288, 8), (20000, 128, 4096, 64)])
def test_long_sums_are_not_cut_off_at_every_step(rows, tile, K, chain):
    """A tensor core cuts sums off towards zero, by half a step on average, 2^-24 of a sum that grows evenly to its end: a
    chain of n such sums is too small by n / 4 steps of 2^-23 on average.  Nothing else is one-sided but what
    the second product cuts off: three parts of a number, one step each."""
    g = torch.Generator().manual_seed(5)
    x = (torch.rand(rows, K, generator=g) + 0.5).to(DEV, torch.bfloat16)
    a = (torch.rand(1, 1, 16, K, generator=g) + 0.5).to(DEV, torch.bfloat16)
    b = torch.eye(16, device=DEV, dtype=torch.bfloat16)[None]
    bank = ops.AdapterBank(a, b, torch.ones(1, device=DEV), (16,))
    ids = torch.zeros(rows, dtype=torch.int32, device=DEV)
    got = ops.adapter_add(torch.zeros(rows, 16, device=DEV), x, bank, ops.adapter_rows(ids, 1, tile))
    some = torch.arange(0, rows, max(1, rows // 512), device=DEV)
    want = x[some].double() @ a[0, 0].double().T
    off = float(((got[some].double() - want) / want).mean())
    assert abs(off) <= (chain / 4 + 3) * 2.0 ** -23, off / 2.0 ** -23
