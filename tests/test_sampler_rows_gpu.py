"""A list of sampling parameters: what a greedy request's other parameters hold is of no account, as it is in one rule for
all."""

import threading

import pytest
import torch

from reflex_b200 import SamplingParams
from reflex_b200.sampling.sampler import Sampler

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("odd", [dict(top_k=-(1 << 40)), dict(top_k=1 << 40), dict(top_p=float("nan")), dict(top_p=-3.0),
                                 dict(min_p=1e300), dict(top_k=0)])
def test_greedy_requests_with_parameters_out_of_range(odd):
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(2, 500, generator=g).to(DEV)
    want = Sampler(SamplingParams(**odd), DEV).pick(logits, [0, 1], [0, 0])
    rules = [SamplingParams(**odd), SamplingParams(temperature=1.0, seed=3, min_p=1.0)]
    assert Sampler(rules, DEV).pick(logits, [0, 1], [0, 0]) == want


def test_what_is_more_than_the_vocabulary_keeps_all():
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(3, 500, generator=g).to(DEV)
    rules = [SamplingParams(temperature=1.0, seed=s, top_k=1 << 40) for s in range(3)]
    none = [SamplingParams(temperature=1.0, seed=s) for s in range(3)]
    assert Sampler(rules, DEV).pick(logits, [0, 1, 2], [0, 1, 2]) == Sampler(none, DEV).pick(logits, [0, 1, 2], [0, 1, 2])


def test_picks_of_two_threads_take_turns_of_their_own():
    """As many picks as a ring has, of another thread, between a pick and the reading of its ids."""
    logits = torch.zeros(2, 500, device=DEV)
    logits[:, 7] = 1.0
    other = torch.zeros(2, 500, device=DEV)
    other[:, 11] = 1.0
    pending = Sampler(SamplingParams(), DEV).pick_async(logits, [0, 1], [0, 0])

    def picks():
        for _ in range(Sampler.RING):
            assert Sampler(SamplingParams(), DEV).pick(other, [0, 1], [0, 0]) == [11, 11]

    t = threading.Thread(target=picks)
    t.start()
    t.join()
    assert pending.wait() == [7, 7] and pending.dev.tolist() == [7, 7]
