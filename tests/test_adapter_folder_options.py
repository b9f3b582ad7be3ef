"""Options of an adapter's folder that leave W -> W + scale B A as it is, and those that do not."""

import json
import os

import pytest

import helpers
from adapter_folders import adapter_folder
from reflex_b200 import UnsupportedArchitecture
from reflex_b200.weights.adapters import read_adapter
from reflex_b200.weights.loader import load_spec
from tiny_configs import ALL


def read(**more):
    folder, pairs = adapter_folder(ALL["A"], 4, 1)
    path = os.path.join(folder, "adapter_config.json")
    with open(path) as f:
        cfg = json.load(f)
    cfg.update(more)
    with open(path, "w") as f:
        json.dump(cfg, f)
    got = read_adapter(folder, load_spec(helpers.model_folder("A", 7, "float32"))[1])
    assert set(got.pairs) == set(pairs) and got.scale == 1.0


@pytest.mark.parametrize("more", [dict(modules_to_save=[]), dict(layer_replication=[]), dict(rank_pattern=None),
                                  dict(alpha_pattern={}), dict(bias="none"), dict(use_dora=None)])
def test_options_that_are_left_off(more):
    read(**more)


@pytest.mark.parametrize("more", [dict(modules_to_save=["embed_tokens"]), dict(layer_replication=[[0, 1]]),
                                  dict(alpha_pattern={"q_proj": 3})])
def test_options_that_change_more(more):
    with pytest.raises(UnsupportedArchitecture, match=next(iter(more))):
        read(**more)


def test_an_adapter_that_begins_at_certain_tokens():
    """Rows before them go without it, which no sequence here does."""
    with pytest.raises(UnsupportedArchitecture, match="alora_invocation_tokens"):
        read(alora_invocation_tokens=[5, 6])
    read(alora_invocation_tokens=None)
