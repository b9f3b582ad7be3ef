"""Captured steps of more sequences than the library's own products take, without adapters and then with them."""

import pytest
import torch

import helpers
import reflex_b200
from adapter_folders import adapter_folder
from reflex_b200 import ops
from tiny_configs import ALL

pytestmark = pytest.mark.gpu
CFG = ALL["B"]


def test_a_large_batch_runs_eagerly_once_with_adapters_too():
    n = ops.GEMV_MAX_ROWS + 6
    model = reflex_b200.Model.load(helpers.model_folder("B", 7, "bfloat16"), max_tokens=(n + 1) * 128)
    model.load_adapters({"a": adapter_folder(CFG, 16, 1)[0]})
    eng = model.engine

    def steps(adapter, count=4):
        seqs = [eng.open(adapter if i % 2 else None) for i in range(n)]
        eng.step([(s, [3 + i], [0]) for i, s in enumerate(seqs)])
        got = [eng.step([(s, [5 + i + t], [0]) for i, s in enumerate(seqs)]).clone() for t in range(count)]
        for s in seqs:
            eng.close(s)
        eng.check_errors()
        return got

    plain = steps(None)
    assert {k[2]: g.graph is not None for k, g in eng._graphs.items()} == {False: True}
    seqs = [eng.open(0 if i % 2 else None) for i in range(n)]
    eng.step([(s, [3 + i], [0]) for i, s in enumerate(seqs)])
    assert [g.graph for k, g in eng._graphs.items() if k[2]] == [None]  # ran eagerly
    for s in seqs:
        eng.close(s)
    captured = steps(0)
    graph, = [g for k, g in eng._graphs.items() if k[2]]
    assert graph.graph is not None and graph.capture_failures == 0
    eng.use_graphs = False
    for got, want in zip(captured, steps(0)):
        assert torch.equal(got, want)
    eng.use_graphs = True
    for got, want in zip(steps(None), plain):
        assert torch.equal(got, want)
