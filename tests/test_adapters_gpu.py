"""Adapters of a step's requests on the GPU: the grouping of the rows and the low-rank products, against a plain
implementation in 64 bits, at the sizes, types and row layouts where they can go wrong."""

import numpy as np
import pytest
import torch

from reflex_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def plain_rows(ids, n, tile):
    key = np.where((ids < 0) | (ids >= n), n, ids)
    order = np.argsort(key, kind="stable")
    counts = np.bincount(key, minlength=n + 1)
    first = np.concatenate([[0], np.cumsum(counts)])
    tiles = [(a, first[a] + i, min(tile, counts[a] - i)) for a in range(n + 1) for i in range(0, counts[a], tile)]
    tiles += [(-1, 0, 0)] * (min(len(ids), n + 1) + len(ids) // tile - len(tiles))
    return order, first, np.array(tiles).reshape(-1, 3)


@pytest.mark.parametrize("tile", [16, 128])
@pytest.mark.parametrize("rows,n,kind", [(1, 1, "any"), (1, 7, "none"), (33, 3, "any"), (64, 64, "own"), (255, 1, "one"),
                                         (256, 1024, "any"), (1000, 5, "runs"), (4097, 500, "any"), (20000, 2, "none"),
                                         (16384, 33, "runs"), (31, 40, "last")])
def test_rows_are_grouped_by_adapter_in_order(rows, n, kind, tile):
    rng = np.random.default_rng(rows + n)
    ids = {"any": lambda: rng.integers(-1, n, rows), "none": lambda: np.full(rows, -1), "own": lambda: rng.permutation(n)[:rows],
           "one": lambda: np.zeros(rows, int), "last": lambda: np.full(rows, n - 1),
           "runs": lambda: np.sort(rng.integers(0, 9, rows)) % (n + 1) - 1}[kind]()
    got = ops.adapter_rows(torch.tensor(ids, dtype=torch.int32, device=DEV), n, tile)
    for g, w in zip((got.order, got.first, got.tiles), plain_rows(ids, n, tile)):
        np.testing.assert_array_equal(g.cpu().numpy(), w)
    ops.check_device_errors(DEV)


def test_adapters_out_of_range_count_as_none_and_are_reported():
    ids = np.array([0, 3, -2, 2, 1 << 30, -1, 1])
    got = ops.adapter_rows(torch.tensor(ids, dtype=torch.int32, device=DEV), 3)
    for g, w in zip((got.order, got.first, got.tiles), plain_rows(ids, 3, 16)):
        np.testing.assert_array_equal(g.cpu().numpy(), w)
    with pytest.raises(ops.CudaError, match="adapter outside its range"):
        ops.check_device_errors(DEV)
    ops.check_device_errors(DEV)


def make(rows, K, cols, rank, n, dtype, out, woven=False, ids=None, ranks=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    N, parts = sum(cols), len(cols)
    x = torch.randn(rows, K, generator=g).to(DEV, dtype)
    base = torch.randn(rows, N, generator=g).to(DEV, out)
    a = torch.randn(n, parts, rank, K, generator=g) * K ** -0.5
    b = torch.randn(n, N, rank, generator=g)
    if ranks is not None:
        used = torch.arange(rank) < torch.tensor(ranks)[:, None]
        a, b = a * used[:, None, :, None], b * used[:, None, :]
    scale = torch.rand(n, generator=g) * 2 - 0.5
    if ids is None:
        ids = torch.randint(-1, n, (rows,), generator=g)
    ids = torch.as_tensor(ids, dtype=torch.int32, device=DEV)
    bank = ops.AdapterBank(a.to(DEV, dtype), b.to(DEV, dtype), scale.to(DEV), cols, woven=woven,
                           ranks=None if ranks is None else torch.tensor(ranks, dtype=torch.int32, device=DEV))
    return base, x, a.to(DEV, dtype), b.to(DEV, dtype), scale.to(DEV), ids, bank


def plain_add(base, x, a, b, scale, ids, cols, woven):
    """The result in 64 bits, and the sum of its terms' magnitudes (what roundings are relative to)."""
    y, size = base.double(), base.double().abs()
    edges = np.cumsum([0] + list(cols))
    for i in range(a.shape[0]):
        r = (ids == i).nonzero()[:, 0]
        for s in range(len(cols)):
            c = slice(s, None, 2) if woven else slice(edges[s], edges[s + 1])
            low = x[r].double() @ a[i, s].double().T
            low_size = x[r].double().abs() @ a[i, s].double().abs().T
            y[r, c] += scale[i].double() * (low @ b[i, c].double().T)
            size[r, c] += scale[i].double().abs() * (low_size @ b[i, c].double().abs().T)
    return y, size


def check(got, base, x, a, b, scale, ids, cols, woven):
    want, size = plain_add(base, x, a, b, scale, ids, cols, woven)
    K, rank = x.shape[1], a.shape[2]
    if x.dtype == torch.float32:
        # a product and a sum per term, eight pieces, the scale and the base: each off by half a step
        inner = (K + 8 + rank + 3) * 2.0 ** -24
    else:
        # sums of 16 products may be cut off, not rounded (a step, 2^-23, each); the low-rank rows go on in two or
        # three bfloat16 parts (2^-17 or better)
        inner = (K / 16 + 64 + rank + 8) * 2.0 ** -23 + 2.0 ** -17
    off = (got.double() - want).abs()
    bound = HALF[got.dtype] * want.abs() * (1 + 2.0 ** -7) + inner * size + 1e-30
    assert bool((off <= bound).all()), float((off / bound).max())
    none = ids < 0
    assert torch.equal(got[none], base[none])


QKV, ONE = (96, 32, 32), (160,)
TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)]


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("rows,K,cols,rank,n,woven", [
    (1, 64, ONE, 16, 1, False), (1, 4096, (512, 128, 128), 16, 4, False), (8, 2048, (256, 256), 16, 8, True),
    (64, 512, QKV, 64, 32, False), (17, 256, (33,), 8, 2, False), (16, 1000, (64, 16, 16), 48, 3, False),
    (5, 999, (7, 3, 2), 5, 2, False), (256, 128, (48, 48), 32, 5, True), (31, 1, (1,), 1, 3, False),
    (3, 40, (5, 5), 3, 2, True), (12, 320, (40, 24, 8, 8, 16), 16, 4, False), (40, 192, (256,), 128, 2, False),
    (257, 256, QKV, 16, 3, False), (700, 1024, (256,), 32, 4, False), (300, 333, (50, 10), 11, 3, False),
    (515, 512, (192, 192), 64, 2, True), (1025, 64, (128,), 128, 1, False), (2000, 128, (130, 2, 64), 16, 700, False),
    (640, 2048, (1000,), 256, 2, False)])
def test_products_beside_the_shared_projection(rows, K, cols, rank, n, woven, dtype, out):
    base, x, a, b, scale, ids, bank = make(rows, K, cols, rank, n, dtype, out, woven)
    got = ops.adapter_add(base, x, bank, ops.adapter_rows(ids, n))
    check(got, base, x, a, b, scale, ids, cols, woven)
    ops.check_device_errors(DEV)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("rows,tile", [(100, 128), (300, 16), (128, 128), (129, 128), (16, 16)])
def test_either_tile_at_any_number_of_rows(rows, tile, dtype, out):
    base, x, a, b, scale, ids, bank = make(rows, 512, QKV, 16, 3, dtype, out, ids=torch.arange(rows) // 7 % 4 - 1)
    got = ops.adapter_add(base, x, bank, ops.adapter_rows(ids, 3, tile))
    check(got, base, x, a, b, scale, ids, QKV, False)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("rows", [9, 400])
def test_adapters_of_smaller_ranks(rows, dtype, out):
    ranks = [64, 8, 0, 1, 33, 16]
    base, x, a, b, scale, ids, bank = make(rows, 256, QKV, 64, 6, dtype, out, ranks=ranks)
    check(ops.adapter_add(base, x, bank, ops.adapter_rows(ids, 6)), base, x, a, b, scale, ids, QKV, False)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("rows", [6, 350])
@pytest.mark.parametrize("woven", [False, True])
def test_in_place_leaves_rows_without_an_adapter_alone(rows, dtype, out, woven):
    cols = (80, 80)
    base, x, a, b, scale, ids, bank = make(rows, 192, cols, 16, 2, dtype, out, woven)
    base[ids < 0] = float("nan")
    before = base.clone()
    got = ops.adapter_add(base, x, bank, ops.adapter_rows(ids, 2), out=base)
    assert got is base
    none = ids < 0
    assert bool(torch.isnan(base[none]).all())
    base[none], before[none] = 0, 0
    check(base, before, x, a, b, scale, ids, cols, woven)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("rows", [7, 290])
@pytest.mark.parametrize("shift,wide", [(0, 8), (1, 3), (4, 12)])
def test_rows_that_lie_apart(rows, dtype, out, shift, wide):
    base, x, a, b, scale, ids, bank = make(rows, 256, QKV, 16, 3, dtype, out)

    def apart(t):
        big = torch.full((rows, t.shape[1] + wide + shift), float("nan"), dtype=t.dtype, device=DEV)
        view = big[:, shift:shift + t.shape[1]]
        view.copy_(t)
        return big, view

    (_, xv), (_, bv), (whole, ov) = apart(x), apart(base), apart(torch.zeros_like(base))
    got = ops.adapter_add(bv, xv, bank, ops.adapter_rows(ids, 3), out=ov)
    check(got.contiguous(), base, x, a, b, scale, ids, QKV, False)
    ov.fill_(float("nan"))
    assert bool(torch.isnan(whole).all())  # nothing beside the rows was written


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("rows", [16, 384])
def test_what_is_not_finite_stays_in_its_row(rows, dtype, out):
    base, x, a, b, scale, ids, bank = make(rows, 512, QKV, 16, 2, dtype, out, ids=torch.arange(rows) % 3 - 1)
    grouped = ops.adapter_rows(ids, 2)
    want = ops.adapter_add(base, x, bank, grouped).clone()
    x[1, 3], x[4, 7], x[0, 0] = float("nan"), float("inf"), float("nan")  # row 0 has no adapter
    got = ops.adapter_add(base, x, bank, grouped)
    touched = torch.zeros(rows, dtype=torch.bool, device=DEV)
    touched[[1, 4]] = True
    assert torch.equal(got[~touched], want[~touched])
    assert bool(torch.isnan(got[1]).all()) and not bool(torch.isfinite(got[4]).any())


@pytest.mark.parametrize("dtype,out", TYPES)
def test_a_row_does_not_depend_on_the_others(dtype, out):
    """The same row alone, in a decode step and among other orders of rows: the same bits."""
    for rows in (64, 500):
        base, x, a, b, scale, ids, bank = make(rows, 768, QKV, 32, 4, dtype, out)
        tile = 16 if rows == 64 else 128
        whole = ops.adapter_add(base, x, bank, ops.adapter_rows(ids, 4, tile))
        perm = torch.randperm(rows, generator=torch.Generator().manual_seed(3)).to(DEV)
        mixed = ops.adapter_add(base[perm], x[perm], bank, ops.adapter_rows(ids[perm], 4, tile))
        assert torch.equal(mixed, whole[perm])
        if dtype == torch.float32:  # the exact path: however the work is cut
            for r in (0, 5, rows - 1):
                one = ops.adapter_add(base[r:r + 1], x[r:r + 1], bank, ops.adapter_rows(ids[r:r + 1], 4, 16))
                assert torch.equal(one[0], whole[r])


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("rows", [24, 600])
def test_captured_steps_replay_with_other_adapters(rows, dtype, out):
    """Grouping and products in a graph: new ids and inputs in the same buffers, and two graphs side by side."""
    graphs = []
    for seed in (1, 2):
        base, x, a, b, scale, ids, bank = make(rows, 256, QKV, 16, 3, dtype, out, seed=seed)
        ops.adapter_add(base, x, bank, ops.adapter_rows(ids, 3))  # sizes what is made once
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.adapter_add(base, x, bank, ops.adapter_rows(ids, 3))
        graphs.append((g, y, base, x, a, b, scale, ids, bank))  # (a graph keeps no memory alive)
    for step in range(3):
        for g, y, base, x, a, b, scale, ids, _ in graphs:
            ids.copy_(torch.randint(-1, 3, (rows,), generator=torch.Generator().manual_seed(step)).to(ids))
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(step)))
        for g, *_ in graphs:
            g.replay()
        for g, y, base, x, a, b, scale, ids, _ in graphs:
            check(y, base, x, a, b, scale, ids, QKV, False)


def test_on_another_stream():
    base, x, a, b, scale, ids, bank = make(32, 512, QKV, 16, 3, torch.bfloat16, torch.float32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.adapter_add(base, x, bank, ops.adapter_rows(ids, 3))
    torch.cuda.current_stream().wait_stream(s)
    check(got, base, x, a, b, scale, ids, QKV, False)


def test_refusals():
    base, x, a, b, scale, ids, bank = make(4, 64, QKV, 16, 2, torch.bfloat16, torch.bfloat16)
    rows = ops.adapter_rows(ids, 2)
    bad = ops.InvalidInput
    with pytest.raises(bad):
        ops.adapter_rows(ids, 0)
    with pytest.raises(bad):
        ops.adapter_rows(ids, 2, tile=64)
    with pytest.raises(bad):
        ops.adapter_rows(ids[:0], 2)
    with pytest.raises(bad):
        ops.adapter_rows(ids.long(), 2)
    with pytest.raises(bad, match="x \\["):
        ops.adapter_add(base, x[:, :32], bank, rows)
    with pytest.raises(bad, match="x is"):
        ops.adapter_add(base, x.float(), bank, rows)
    with pytest.raises(bad, match="grouped"):
        ops.adapter_add(base, x, bank, ops.adapter_rows(ids, 3))
    with pytest.raises(bad, match="grouped"):
        ops.adapter_add(base[:3], x[:3], bank, rows)
    with pytest.raises(bad, match="base is"):
        ops.adapter_add(base.half(), x, bank, rows)
    with pytest.raises(bad, match="like base"):
        ops.adapter_add(base, x, bank, rows, out=base.float())
    with pytest.raises(bad, match="side by side"):
        ops.adapter_add(base, x.t().contiguous().t(), bank, rows)
    with pytest.raises(bad, match="do not overlap"):
        ops.adapter_add(base, x[:1].expand(4, -1), bank, rows)
    with pytest.raises(bad, match="woven"):
        ops.AdapterBank(a, b, scale, QKV, woven=True)
    with pytest.raises(bad, match="fit"):
        ops.AdapterBank(a, b, scale, (96, 64))
    with pytest.raises(bad):
        ops.AdapterBank(a, b.float(), scale, QKV)
    with pytest.raises(bad):
        ops.AdapterBank(a, b, scale[:1], QKV)


def test_a_result_that_overlaps_what_is_read():
    base, x, a, b, scale, ids, bank = make(4, 160, QKV, 16, 2, torch.bfloat16, torch.bfloat16)
    rows = ops.adapter_rows(ids, 2)
    wide = torch.zeros(8, 160, dtype=torch.bfloat16, device=DEV)
    wide[::2] = base
    for out, was in ((x, base), (wide[1:5], wide[:4]), (wide[:4], wide[::2])):
        with pytest.raises(ops.InvalidInput, match="overlaps"):
            ops.adapter_add(was, x, bank, rows, out=out)
    both = torch.zeros(4, 320, dtype=torch.bfloat16, device=DEV)  # side by side in the same rows is no overlap
    both[:, :160] = base
    ops.adapter_add(both[:, :160], x, bank, rows, out=both[:, 160:])
    check(both[:, 160:].contiguous(), base, x, a, b, scale, ids, QKV, False)
    view = base.view(4, 160)  # base itself by another tensor
    before = base.clone()
    check(ops.adapter_add(base, x, bank, rows, out=view), before, x, a, b, scale, ids, QKV, False)
