"""Adapters on the host: what a folder has to hold, how prompts get theirs, and sampling parameters a prompt."""

import json
import os

import pytest
import torch

import helpers
from adapter_folders import adapter_folder
from reflex_b200 import CheckpointError, InvalidInput, IoError, SamplingParams, UnsupportedArchitecture, ops
from reflex_b200.engine.generate import generate
from reflex_b200.weights import write_safetensors
from reflex_b200.weights.adapters import read_adapter
from reflex_b200.weights.loader import load_spec
from tiny_configs import ALL

CFG = ALL["A"]


def spec():
    return load_spec(helpers.model_folder("A", 7, "float32"))[1]


def change(folder, **more):
    path = os.path.join(folder, "adapter_config.json")
    with open(path) as f:
        cfg = json.load(f)
    cfg.update(more)
    with open(path, "w") as f:
        json.dump(cfg, f)


def test_a_folder_is_read():
    folder, pairs = adapter_folder(CFG, 4, 1, alpha=6)
    got = read_adapter(folder, spec())
    assert got.scale == 1.5 and set(got.pairs) == set(pairs)
    for name, (a, b) in pairs.items():
        assert torch.equal(got.pairs[name][0], a) and torch.equal(got.pairs[name][1], b)
    change(folder, use_rslora=True)
    assert read_adapter(folder, spec()).scale == 3.0


@pytest.mark.parametrize("more,error", [
    (dict(r=0), CheckpointError), (dict(r="4"), CheckpointError), (dict(lora_alpha=None), CheckpointError),
    (dict(lora_alpha=float("nan")), CheckpointError), (dict(r=8), CheckpointError), (dict(use_dora=True), UnsupportedArchitecture),
    (dict(bias="all"), UnsupportedArchitecture), (dict(rank_pattern={"q_proj": 2}), UnsupportedArchitecture),
    (dict(modules_to_save=["lm_head"]), UnsupportedArchitecture)])
def test_configurations_that_do_not_fit(more, error):
    folder, _ = adapter_folder(CFG, 4, 1)
    change(folder, **more)
    with pytest.raises(error):
        read_adapter(folder, spec())


def test_tensors_that_do_not_fit():
    H = CFG["hidden_size"]
    name = "base_model.model.model.layers.0.self_attn.q_proj"
    good = [(name + ".lora_A.weight", torch.zeros(4, H)),
            (name + ".lora_B.weight", torch.zeros(CFG["num_attention_heads"] * CFG["head_dim"], 4))]
    for tensors, word in ((good[:1], "lora_B is missing"), ([], "no adapter tensors"),
                          (good + [("base_model.model.model.layers.99.self_attn.q_proj.lora_A.weight", torch.zeros(4, H))], "no matrix"),
                          (good + [("base_model.model.model.norm.lora_A.weight", torch.zeros(4, H))], "no matrix"),
                          ([(good[0][0], torch.zeros(4, H + 1)), good[1]], "expected"),
                          ([(good[0][0], torch.zeros(4, H, dtype=torch.int32)), good[1]], "expected")):
        folder, _ = adapter_folder(CFG, 4, 1, layers=[0], roles=("self_attn.q_proj",))
        write_safetensors(os.path.join(folder, "adapter_model.safetensors"), tensors)
        with pytest.raises(CheckpointError, match=word):
            read_adapter(folder, spec())
    with pytest.raises(IoError):
        read_adapter("/nowhere", spec())


class Slots:
    held_count = 0


class FakeEngine:
    """Every token is the one before plus one; it remembers which adapter a sequence was opened with."""

    class cache:
        max_positions, max_tokens, max_slots, slots = 1000, 10000, 8, Slots()

    def __init__(self):
        self.opened, self.next = [], 0

    def open(self, adapter=None):
        self.opened.append(adapter)
        self.next += 1
        return self.next

    def close(self, seq):
        pass

    def step(self, entries):
        return [t[w[0]] + 1 for _, t, w in entries]


def test_prompts_get_their_adapters_and_their_stop_tokens():
    e = FakeEngine()
    out = generate(e, [[1], [10], [20]], 5, lambda l, r, s: l, stop_token_ids=[3], stops_of=[(), (12,), ()],
                   adapters=[None, 1, 0])
    assert out == [[2, 3], [11, 12], [21, 22, 23, 24, 25]]
    assert e.opened == [None, 1, 0]


def test_min_p_is_checked():
    SamplingParams(temperature=1.0, min_p=0.1).validate()
    SamplingParams(min_p=7.0).validate()  # ignored when greedy
    for bad in (-0.1, 1.1, float("nan")):
        with pytest.raises(InvalidInput, match="min_p"):
            SamplingParams(temperature=1.0, min_p=bad).validate()


@pytest.mark.parametrize("text", ["[1, 2]", "7", '{"r": 4, "lora_alpha": 1%s}' % ("0" * 400)])
def test_configurations_that_are_no_object_or_out_of_range(text):
    folder, _ = adapter_folder(CFG, 4, 1)
    with open(os.path.join(folder, "adapter_config.json"), "w") as f:
        f.write(text)
    with pytest.raises(CheckpointError):
        read_adapter(folder, spec())


def test_rows_in_tiles_that_no_kernel_has():
    n = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(InvalidInput, match="16 or 128"):
        ops.AdapterRows(n, n, n.view(2, 2), 32)
    for order, first, tiles in ((n, n, n.view(2, 2)), (n.view(2, 2), n, n[:3].view(1, 3)), (n, n[:2], n[:3].view(1, 3))):
        with pytest.raises(InvalidInput, match="order"):
            ops.AdapterRows(order, first, tiles, 16)


def test_sampling_needs_a_temperature_and_a_number_a_row():
    one = torch.ones(2)
    for t, u in ((None, one), (one, None)):
        with pytest.raises(InvalidInput, match="temperature"):
            ops.sample_rows(torch.zeros(2, 5), t, u)


def test_what_overlaps():
    big = torch.zeros(6, 20)
    for a, b, want in ((big[:, :8], big[:, 8:], False), (big[:, 8:], big[:, :8], False), (big[:, :9], big[:, 8:], True),
                       (big[:3], big[3:], False), (big[:4, :8], big[2:, :8], True), (big[:4, :8], big[2:, 8:16], False),
                       (big[1:, 12:], big[:5, :12], False), (big, big[2:3, 4:5], True), (big[:, :4], big.view(3, 40)[:, 4:8], True),
                       (big, big.clone(), False), (big[:, :8], big.view(torch.int16).view(6, 40)[:, 16:], False)):
        assert ops._overlap(a, b) is want
