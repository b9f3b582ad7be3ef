"""Adapters belong to the weights: several engines of one model see each other's open sequences and captured steps."""

import pytest
import torch

import helpers
from reflex_b200 import InvalidInput, Model
from reflex_b200.engine import Engine
from reflex_b200.engine.model import CausalLM
from reflex_b200.weights.loader import load_spec


def two():
    lm = CausalLM(load_spec(helpers.model_folder("A", 7, "float32"))[1], torch.float32, "cpu")
    return lm, Engine(lm, max_tokens=256), Engine(lm, max_tokens=256)


def test_no_exchange_while_another_engine_has_a_sequence_open():
    lm, one, other = two()
    lm.n_adapters = 1
    s = other.open(0)
    with pytest.raises(InvalidInput, match="open"):
        one.load_adapters([])
    other.close(s)
    one.load_adapters([])
    assert lm.n_adapters == 0
    with pytest.raises(InvalidInput):
        other.open(0)


def test_steps_that_another_engine_captured_go():
    lm, one, other = two()
    for e in (one, other):
        e._graphs = {(1, 256, True): object(), (1, 256, False): "plain"}
    one.load_adapters([])
    assert one._graphs == other._graphs == {(1, 256, False): "plain"}


def test_an_engine_that_is_gone_does_not_count():
    lm, one, other = two()
    lm.n_adapters = 1
    other.open(0)
    del other
    one.load_adapters([])


def test_names_are_the_weights_own():
    lm, _, _ = two()
    first, second = Model(lm, max_tokens=256), Model(lm, max_tokens=256)
    first.engine.load_adapters([], ["x", "y"])  # (as `Model.load_adapters` does with what it has read)
    assert first.adapter_names == second.adapter_names == ["x", "y"] and second.adapter("y") == 1
    second.engine.load_adapters([])
    assert first.adapter_names == []
    with pytest.raises(InvalidInput, match="no adapter"):
        first.adapter("x")
