"""A token a row with the row's own temperature, top-k, top-p and min-p, against a plain sampler in 64 bits that is
given the same uniform numbers."""

import math

import numpy as np
import pytest
import torch

from reflex_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def plain_token(l, T, u, k=0, p=1.0, m=0.0):
    """The definition, in 64 bits; l float32, the rules as the kernel gets them (32-bit numbers)."""
    l = np.where(np.isnan(l), -np.inf, l.astype(np.float64))
    top = l.max()
    if top == -np.inf:
        return 0
    if not T > 0:
        return int(np.flatnonzero(l == top)[-1])
    with np.errstate(invalid="ignore"):
        e = np.where(l == top, 1.0, np.exp((l - top) / T) if np.isfinite(top) else 0.0)
    order = np.argsort(-l, kind="stable")
    down = e[order]
    before = np.concatenate([[0.0], np.cumsum(down)[:-1]])
    keep = down > 0
    if 0 < k < len(l):
        keep &= np.arange(len(l)) < k
    if p < 1:
        keep &= before < max(p, 0.0) * down.sum()
    if m > 0:
        keep &= down >= min(m, 1.0)
    keep[0] = True
    kept = np.zeros_like(e)
    kept[order[keep]] = down[keep]
    sums = np.cumsum(kept)
    return int(np.flatnonzero((sums >= u * sums[-1]) & (kept > 0))[0])


def run(logits, T, u, k=None, p=None, m=None):
    f = lambda v, t: None if v is None else torch.tensor(np.asarray(v), dtype=t, device=DEV)  # noqa: E731
    l = logits if isinstance(logits, torch.Tensor) else torch.tensor(logits, device=DEV)
    return ops.sample_rows(l, f(T, torch.float32), f(u, torch.float32), f(k, torch.int32), f(p, torch.float32),
                           f(m, torch.float32)).tolist()


def check(logits, T, u, k=None, p=None, m=None, at=None):
    B = len(logits)
    got = run(logits if at is None else at, T, u, k, p, m)
    f32 = lambda v: [float(np.float32(x)) for x in v]  # noqa: E731
    want = [plain_token(logits[b], f32(T)[b], f32(u)[b], 0 if k is None else k[b], 1.0 if p is None else f32(p)[b],
                        0.0 if m is None else f32(m)[b]) for b in range(B)]
    assert got == want


def rows(B, V, spread, seed):
    rng = np.random.default_rng(seed)
    l = rng.normal(0, spread, (B, V)).astype(np.float32)
    if V > 20:
        l[:, rng.integers(0, V, 5)] += np.float32(3 * spread)
    return l, rng


@pytest.mark.parametrize("V", [1, 2, 5, 127, 4096, 4099, 32003, 151936, 300001])
@pytest.mark.parametrize("cuts", ["none", "k", "p", "m", "kpm"])
@pytest.mark.parametrize("spread", [0.3, 2.0, 8.0])
def test_tokens_against_the_plain_sampler(V, cuts, spread):
    B = 5
    l, rng = rows(B, V, spread, V)
    T = rng.uniform(0.3, 1.5, B)
    u = np.floor(rng.uniform(0, 1, B) * 2 ** 24) / 2 ** 24
    k = [1, 2, 40, 1000, V] if "k" in cuts else None
    p = [0.0, 0.3, 0.9, 0.999, 1.0] if "p" in cuts else None
    m = [1.0, 0.5, 0.1, 1e-4, 0.0] if "m" in cuts else None
    if cuts == "kpm":
        k, p, m = [50, 0, 3, -1, 500], [0.95, 0.9, 2.0, 0.5, 1.0], [0.01, 0.2, 0.0, 0.0, 0.05]
    check(l, T, u, k, p, m)


def test_every_row_has_its_own_rules():
    B = 64
    l, rng = rows(B, 50000, 2.5, 1)
    l[rng.uniform(size=l.shape) < 0.4] = -np.inf
    T = np.where(rng.uniform(size=B) < 0.2, 0.0, rng.uniform(0.2, 2, B))
    T[3], T[4] = np.nan, -1.0
    check(l, T, np.floor(rng.uniform(0, 1, B) * 2 ** 24) / 2 ** 24, [int(v) for v in rng.integers(-1, 80, B)],
          list(rng.uniform(0.2, 1.2, B)), list(rng.uniform(-0.05, 0.3, B)))


@pytest.mark.parametrize("V", [7, 5000, 151936, 500000])
def test_ties_are_kept_lowest_index_first(V):
    """Few distinct logits: the cut falls among equals, which also straddle the row's pieces."""
    rng = np.random.default_rng(V)
    l = rng.integers(0, 3, (8, V)).astype(np.float32) - 1
    l[0], l[1] = 0.0, -0.0
    l[1, ::2] = 0.0
    u = [0.0, 0.999999, 0.5, 0.25, 0.75, 0.1, 0.9, 0.333]
    some = max(1, V // 3)
    check(l, [0.7] * 8, u, [some, some, V - 1, some + 1, 5, 1, V, 0], [1.0, 1.0, 1.0, 0.5, 1.0, 1.0, 0.37, 0.61])
    check(l, [0.7] * 8, u, None, [0.5, 0.1, 0.999, 0.0, 0.2, 0.4, 0.6, 0.8])


def test_what_is_masked_is_never_picked():
    V = 9000
    l, rng = rows(12, V, 1.0, 5)
    only = [3, 4095, 4096, 8999]
    for r, i in enumerate(only):  # one token left
        l[r] = -np.inf
        l[r, i] = -1e30
    l[4, :] = -np.inf                      # nothing left
    l[5, :] = np.nan
    l[6, ::2], l[6, 1::2] = np.nan, -np.inf
    l[7, 100:] = np.finfo(np.float32).min  # the type's lowest value is no mask: it is a small logit
    l[8, 50], l[8, 7000] = np.inf, np.inf  # they share everything
    l[9, 1::3] = np.nan
    l[10] = np.finfo(np.float32).min       # all alike
    l[11, :] = np.finfo(np.float32).max
    for u in (0.0, 0.4, 0.51, 0.9999):
        for T in (0.0, 0.8, 1e-30, 1e30):
            check(l, [T] * 12, [u] * 12)
            check(l, [T] * 12, [u] * 12, [3] * 12, [0.7] * 12, [0.2] * 12)


def test_edges_of_the_uniform_number_and_the_cuts():
    l = np.log(np.array([[0.5, 0.25, 0.25]], dtype=np.float32))
    V = 3
    for u, want in ((0.0, 0), (0.25, 0), (0.6, 1), (0.9999, 2)):
        assert run(l, [1.0], [u]) == [want]
    assert run(l, [1.0], [0.9999], k=[2]) == [1]
    assert run(l, [1.0], [0.9999], p=[0.4]) == [0]
    assert run(l, [1.0], [0.9999], m=[0.9]) == [0]
    assert run(l, [1.0], [0.9999], m=[7.0]) == [0]           # above one: the most probable alone
    nan = float("nan")
    assert run(l, [1.0], [0.9999], p=[nan], m=[nan]) == [V - 1]   # no rule


def test_rows_that_lie_apart_and_unaligned():
    l, rng = rows(6, 40001, 2.0, 9)
    for shift, wide in ((0, 3), (1, 0), (4, 4)):
        big = torch.full((6, 40001 + shift + wide), 1e9, device=DEV)
        view = big[:, shift:shift + 40001]
        view.copy_(torch.tensor(l))
        check(l, [0.9] * 6, [0.1, 0.3, 0.5, 0.7, 0.9, 0.99], [50] * 6, [0.9] * 6, [0.01] * 6, at=view)


def test_many_rows_and_replays():
    """More rows than the device holds clusters; a captured draw follows its buffers; runs agree to the bit."""
    B, V = 1500, 20000
    l, rng = rows(B, V, 2.0, 11)
    T, u = rng.uniform(0.5, 1.5, B).astype(np.float32), np.floor(rng.uniform(0, 1, B) * 2 ** 24).astype(np.float32) / 2 ** 24
    some = rng.choice(B, 40, replace=False)
    got = run(l, T, u, p=[0.9] * B)
    assert run(l, T, u, p=[0.9] * B) == got
    for b in some:
        assert got[b] == plain_token(l[b], float(T[b]), float(u[b]), 0, float(np.float32(0.9)))
    logits, out = torch.tensor(l[:4], device=DEV), torch.empty(4, dtype=torch.int32, device=DEV)
    t, uu = torch.tensor(T[:4], device=DEV), torch.tensor(u[:4], device=DEV)
    ops.sample_rows(logits, t, uu, out=out)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        ops.sample_rows(logits, t, uu, out=out)
    for i in (4, 8):
        logits.copy_(torch.tensor(l[i:i + 4]))
        t.copy_(torch.tensor(T[i:i + 4]))
        g.replay()
        assert out.tolist() == [plain_token(l[i + j], float(T[i + j]), float(u[j])) for j in range(4)]


def test_agrees_with_the_sampler_of_one_rule_for_all():
    """Peaked rows and cuts that leave few borders: `sample`, which has no min-p, picks the same tokens."""
    B, V = 32, 30000
    l, rng = rows(B, V, 4.0, 13)
    u = torch.tensor(np.floor(rng.uniform(0, 1, B) * 2 ** 24) / 2 ** 24, dtype=torch.float32, device=DEV)
    logits, T = torch.tensor(l, device=DEV), torch.full((B,), 0.8, device=DEV)
    k, p = torch.full((B,), 40, dtype=torch.int32, device=DEV), torch.full((B,), 0.95, device=DEV)
    assert torch.equal(ops.sample(logits, T, u, top_k=k, top_p=p), ops.sample_rows(logits, T, u, top_k=k, top_p=p))
    assert torch.equal(ops.argmax(logits), ops.sample_rows(logits, T * 0, u))


def test_refusals():
    l, T, u = torch.zeros(2, 10, device=DEV), torch.ones(2, device=DEV), torch.zeros(2, device=DEV)
    bad = ops.InvalidInput
    for call in (lambda: ops.sample_rows(l.double(), T, u), lambda: ops.sample_rows(l, T[:1], u),
                 lambda: ops.sample_rows(l, T, u, top_k=T), lambda: ops.sample_rows(l, T, u, top_p=u.double()),
                 lambda: ops.sample_rows(l, T, u, out=torch.zeros(2, device=DEV)), lambda: ops.sample_rows(l[:0], T[:0], u[:0]),
                 lambda: ops.sample_rows(l[:, :0], T, u), lambda: ops.sample_rows(l[0], T, u),
                 lambda: ops.sample_rows(l.t().contiguous().t(), T, u), lambda: ops.sample_rows(l, T, u, min_p=T[:1])):
        with pytest.raises(bad):
            call()
    with pytest.raises(ops.CudaError):
        ops.sample_rows(l.cpu(), T, u)
    with pytest.raises(ops.CudaError):
        ops.sample_rows(l, T.cpu(), u)


@pytest.mark.parametrize("B", [2, 6, 70])  # clusters of 16, of 8, and two CTAs an SM
@pytest.mark.parametrize("many", [60, 130, 200, 270, 512, 513, 1000, 1025, 3000])
def test_a_cut_among_many_entries_of_a_bin(many, B):
    """So many logits within an eighth of 1/32 octave, a third of them of a few equal values, and the cut among them."""
    V = 40000
    rng = np.random.default_rng(many + B)
    l = np.full((B, V), -12.0, np.float32) + rng.uniform(0, 1, (B, V)).astype(np.float32)
    for b in range(B):
        at = rng.permutation(V)[:many + 3]
        near = rng.uniform(-2.0, -1.9973, many).astype(np.float32)
        near[: many // 3] = near[rng.integers(0, 7, many // 3)]
        l[b, at] = np.concatenate([near, np.float32([0.0, 0.1, 0.2])])
    u = np.floor(rng.uniform(0, 1, B) * 2 ** 24) / 2 ** 24
    check(l, [1.0] * B, u, [int(v) for v in rng.integers(4, many + 3, B)])
    check(l, [1.0] * B, u, None, list(rng.uniform(0.3, 0.95, B)))
    check(l, [1.0] * B, u, [int(v) for v in rng.integers(4, many + 3, B)], list(rng.uniform(0.3, 0.95, B)), [0.05] * B)
