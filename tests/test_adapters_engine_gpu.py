"""Requests with adapters and sampling rules of their own through the entry points: against the plain model with the
adapter merged into its weights, in batches, in captured steps, from the command line."""

import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import helpers
import plain_model as pm
import reflex_b200
from adapter_folders import adapter_folder, merged
from reflex_b200 import InvalidInput, SamplingParams, UnsupportedArchitecture
from tiny_configs import ALL

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAME = "B"
CFG = ALL[NAME]


def loaded(weights, **kw):
    folder = helpers.model_folder(NAME, 7, "float32" if weights == "f32" else "bfloat16")
    made = {"all": adapter_folder(CFG, 8, 1, alpha=12), "attention": adapter_folder(CFG, 16, 2, roles=("self_attn.q_proj", "self_attn.v_proj")),
            "one": adapter_folder(CFG, 3, 3, roles=("mlp.down_proj", "mlp.up_proj"), layers=[1])}
    model = reflex_b200.Model.load(folder, weights=weights, max_tokens=8192, **kw)
    model.load_adapters({n: f for n, (f, _) in made.items()})
    cfg, w = pm.read_model(folder)
    plain = {n: merged(w, pairs, 1.5 if n == "all" else 1.0) for n, (_, pairs) in made.items()}
    plain[None] = w
    return model, cfg, plain


NAMES = (None, "all", "attention", "one", "all", None, "one")


def prompts():
    return [helpers.random_tokens(n, CFG["vocab_size"], 60 + n) for n in (5, 33, 64, 1, 100, 17, 130)]


@pytest.mark.parametrize("weights", ["f32", "bf16"])
def test_a_mixed_batch_against_merged_weights(weights):
    """Prompts of unequal length with different adapters in one step, then single tokens of all of them."""
    model, cfg, plain = loaded(weights)
    eng = model.engine
    ps = prompts()
    seqs = [eng.open(None if n is None else model.adapter(n)) for n in NAMES]
    limit = 1e-4 if weights == "f32" else 3e-2  # the limits that the model is held to without adapters
    try:
        logits = eng.step([(s, p, [len(p) - 1]) for s, p in zip(seqs, ps)]).cpu().numpy()
        for step in range(4):
            for row, (p, n) in enumerate(zip(ps, NAMES)):
                off = {m: helpers.rel_err(logits[row], pm.forward(cfg, plain[m], p)[-1]) for m in plain}
                assert off[n] < limit, (step, row, n)
                # and it is this adapter's model that the row is nearest to
                assert all(off[m] > 1.5 * off[n] for m in plain if m != n), (step, row, n, off)
            nxt = [(7 * step + 3 * i) % cfg["vocab_size"] for i in range(len(ps))]
            ps = [p + [t] for p, t in zip(ps, nxt)]
            logits = eng.step([(s, [t], [0]) for s, t in zip(seqs, nxt)]).cpu().numpy()
        eng.check_errors()
    finally:
        for s in seqs:
            eng.close(s)


def test_exact_rows_do_not_depend_on_the_batch():
    """In 32-bit: alone, among others, in chunks: the same bits."""
    model, _, _ = loaded("f32")
    eng = model.engine
    ps = prompts()
    seqs = [eng.open(None if n is None else model.adapter(n)) for n in NAMES]
    together = eng.step([(s, p, [len(p) - 1]) for s, p in zip(seqs, ps)]).clone()
    for s in seqs:
        eng.close(s)
    for i, (p, n) in enumerate(zip(ps, NAMES)):
        s = eng.open(None if n is None else model.adapter(n))
        cut = len(p) // 2
        if cut:
            eng.step([(s, p[:cut], [])])
        alone = eng.step([(s, p[cut:], [len(p) - cut - 1])])
        eng.close(s)
        assert torch.equal(alone[0], together[i]), (i, n)


@pytest.mark.parametrize("batch", [1, 7])
def test_captured_steps_with_adapters(batch):
    """A graph of steps with adapters follows sequences with other adapters; steps without any keep their own graph
    and their results."""
    eager, _, _ = loaded("bf16", use_graphs=False)
    model, _, _ = loaded("bf16")
    ps, outs = prompts()[:batch], []
    for names in (NAMES[:batch], [None] * batch, (NAMES[1:] + NAMES[:1])[:batch]):
        names = list(names)
        got = [m.generate(ps, 10, adapters=names) for m in (eager, model)]
        assert got[0] == got[1], names
        outs.append(got[0])
    keys = list(model.engine._graphs)
    assert {k[2] for k in keys} == {False, True}
    base = reflex_b200.Model.load(helpers.model_folder(NAME, 7, "bfloat16"), max_tokens=8192)
    assert base.generate(ps, 10) == outs[1]


@pytest.mark.parametrize("weights", ["f32", "bf16"])
def test_requests_with_their_own_adapters_and_rules_together(weights):
    """One generate call of everything: what a request gets does not depend on what shares its batch, greedy requests
    get what a greedy call gives, and min-p and stop tokens are each request's own."""
    model, _, _ = loaded(weights, max_batch=7)
    ps = prompts()
    rules = [SamplingParams(), SamplingParams(temperature=0.8, seed=3, top_k=20), SamplingParams(temperature=1.1, seed=4, min_p=0.05),
             SamplingParams(temperature=0.9, seed=5, top_p=0.8, min_p=0.01), SamplingParams(temperature=1.5, seed=6),
             SamplingParams(temperature=float("nan")), SamplingParams(temperature=1.0, seed=7, min_p=1.0)]
    got = model.generate(ps, 12, rules, adapters=list(NAMES))
    assert model.last_stats.batches == 1
    assert got == model.generate(ps, 12, rules, adapters=list(NAMES))
    greedy = model.generate(ps, 12, adapters=list(NAMES))
    for i in (0, 5, 6):  # min_p = 1 leaves the most probable alone
        assert got[i] == greedy[i]
    assert got != greedy
    if weights == "f32":  # bits that do not depend on the batch: neither do the tokens
        model.max_batch = 2
        assert model.generate(ps, 12, rules, adapters=list(NAMES)) == got
        model.decode_ahead = False
        assert model.generate(ps, 12, rules, adapters=list(NAMES)) == got
    stop = got[4][3]
    rules[4] = SamplingParams(temperature=1.5, seed=6, stop_token_ids=(stop,))
    again = model.generate(ps, 12, rules, adapters=list(NAMES))
    first = got[4].index(stop)
    assert again[4] == got[4][:first + 1]
    if weights == "f32":
        assert [again[i] for i in (0, 1, 2, 3, 5, 6)] == [got[i] for i in (0, 1, 2, 3, 5, 6)]


def test_one_rule_for_all_with_min_p():
    model, _, _ = loaded("f32")
    ps = prompts()[:4]
    got = model.generate(ps, 8, SamplingParams(temperature=0.9, seed=11, min_p=0.1, top_k=30))
    assert got == model.generate(ps, 8, [SamplingParams(temperature=0.9, seed=11, min_p=0.1, top_k=30)] * 4)
    assert model.generate(ps, 8, SamplingParams(temperature=0.9, seed=11, min_p=1.0)) == model.generate(ps, 8)


def test_adapters_are_exchanged_and_refused():
    model, cfg, plain = loaded("f32")
    eng, p = model.engine, prompts()[1]
    with pytest.raises(InvalidInput, match="no adapter"):
        model.generate([p], 1, adapters="other")
    with pytest.raises(InvalidInput, match="as many adapters"):
        model.generate([p, p], 1, adapters=["all"])
    with pytest.raises(InvalidInput, match="as many sampling"):
        model.generate([p, p], 1, [SamplingParams()])
    with pytest.raises(InvalidInput):
        eng.open(3)
    held = eng.cache.slots.held_count
    s = eng.open(0)
    with pytest.raises(InvalidInput, match="open"):
        model.load_adapters({})
    eng.close(s)
    assert eng.cache.slots.held_count == held
    # a matrix whose part takes no adapters: refused whole, what was loaded stays
    before = model.generate(p, 3, adapters="all")
    H, V = CFG["hidden_size"], CFG["vocab_size"]
    from reflex_b200.weights.adapters import Adapter

    with pytest.raises(UnsupportedArchitecture):
        eng.load_adapters([Adapter(1.0, {"model.embed_tokens.weight": (torch.zeros(2, H), torch.zeros(V, 2))})])
    assert model.generate(p, 3, adapters="all") == before
    # others in their place
    folder, pairs = adapter_folder(CFG, 40, 9)
    model.load_adapters({"new": folder})
    s = eng.open(model.adapter("new"))
    got = eng.step([(s, p, [len(p) - 1])]).cpu().numpy()[0]
    eng.close(s)
    assert helpers.rel_err(got, pm.forward(cfg, merged(plain[None], pairs), p)[-1]) < 2e-4
    model.load_adapters({})
    with pytest.raises(InvalidInput):
        model.generate(p, 1, adapters="new")
    assert model.generate(p, 3) == reflex_b200.Model.load(helpers.model_folder(NAME, 7, "float32"), weights="f32",
                                                          max_tokens=1024).generate(p, 3)


def test_other_designs_refuse_adapters():
    from purusun_models import model_folder  # its attention has options that go without

    folder = model_folder("A")
    model = reflex_b200.Model.load(folder, weights="f32", max_tokens=1024)
    from reflex_b200.engine.model import expected_tensors
    from reflex_b200.weights.adapters import Adapter

    for name, (where, info) in expected_tensors(model.spec).items():
        if info.role == "matrix" and len(where) == 4:
            out, width = info.concrete_shape()
            with pytest.raises(UnsupportedArchitecture):
                model.engine.load_adapters([Adapter(1.0, {name: (torch.zeros(2, width), torch.zeros(out, 2))})])


def test_command_line():
    folder = helpers.model_folder(NAME, 7, "float32")
    dirs = [adapter_folder(CFG, 8, s)[0] for s in (1, 2)]
    args = [sys.executable, os.path.join(ROOT, "bin", "reflex"), "generate", folder, "1,2,3", "--prompt-ids", "4,5", "--max-tokens",
            "6", "--weights", "f32", "--json"]

    def run(*more):
        r = subprocess.run(args + list(more), capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr
        return [json.loads(l)["token_ids"] for l in r.stdout.strip().splitlines()]

    model = reflex_b200.Model.load(folder, weights="f32", max_tokens=1024)
    model.load_adapters({"a": dirs[0], "b": dirs[1]})
    ps = [[1, 2, 3], [4, 5]]
    assert run("--adapter", dirs[0], "--adapter", dirs[1]) == model.generate(ps, 6, adapters=["a", "b"])
    assert run("--adapter", "-", "--adapter", dirs[1]) == model.generate(ps, 6, adapters=[None, "b"])
    assert run("--adapter", dirs[0], "--temperature", "0.9", "--seed", "5", "--min-p", "0.1") == model.generate(
        ps, 6, SamplingParams(temperature=0.9, seed=5, min_p=0.1), adapters="a")
