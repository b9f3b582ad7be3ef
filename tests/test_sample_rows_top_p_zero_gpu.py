"""A top-p of nothing keeps the most probable token alone, the lowest index among equals, however many logits lie beside
it."""

import numpy as np
import pytest
import torch

from reflex_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("B", [2, 6, 70])
@pytest.mark.parametrize("many", [2, 3, 60, 512, 600, 1024, 2000])
@pytest.mark.parametrize("kind", ["near", "equal", "both"])
def test_the_first_token_alone(B, many, kind):
    V = 40000
    rng = np.random.default_rng(many + B)
    l = rng.uniform(-12.0, -11.0, (B, V)).astype(np.float32)
    want = []
    for b in range(B):
        at = rng.permutation(V)[:many]
        top = rng.uniform(-0.005, 0.0, many).astype(np.float32)
        if kind != "near":
            top[: many if kind == "equal" else (many + 1) // 2] = 0.0
        l[b, at] = top
        want.append(int(np.argmax(l[b])))
    logits = torch.tensor(l, device=DEV)

    def full(v, t=torch.float32):
        return torch.full((B,), v, dtype=t, device=DEV)

    for p in (0.0, -0.5, 1e-30):
        for u in (0.0, 0.3, 0.7, 0.9999999):
            for k, m in ((None, None), (full(many, torch.int32), None), (full(1, torch.int32), full(0.001)), (None, full(0.5))):
                out = full(-1, torch.int32)
                ops.sample_rows(logits, full(1.0), full(u), top_k=k, top_p=full(p), min_p=m, out=out)
                assert out.tolist() == want, (p, u)


def test_as_the_sampler_of_one_rule_for_all():
    """Two equal maxima: rows of a list of rules and `sample` alike."""
    l = torch.full((3, 9), -4.0, device=DEV)
    l[:, 2], l[:, 6] = 1.0, 1.0
    one = torch.ones(3, device=DEV)
    u = torch.tensor([0.0, 0.6, 0.999], device=DEV)
    assert ops.sample_rows(l, one, u, top_p=one * 0).tolist() == ops.sample(l, one, u, top_p=one * 0).tolist() == [2, 2, 2]
