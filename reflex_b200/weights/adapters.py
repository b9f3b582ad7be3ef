"""Low-rank adapters from a folder: adapter_config.json and adapter_model.safetensors.

An adapter changes some of a model's matrices, W -> W + scale B A, A [r, in] and B [out, r].  The files are those that
the usual training tools write: the module's name under `base_model.model.`, `.lora_A.weight` and `.lora_B.weight`
behind it; scale = lora_alpha / r (lora_alpha / sqrt(r) with `use_rslora`).  (The reference merges one adapter into the
weights when it loads them, src/lora.rs; here any number stays beside the shared weights and every sequence has its
own.)
"""

from __future__ import annotations

import json
import math
import os
from dataclasses import dataclass
from typing import Dict, Tuple

import torch

from ..config.spec import ModelSpec
from ..errors import CheckpointError, IoError, UnsupportedArchitecture
from .safetensors_io import SafetensorsFile

PREFIX = "base_model.model."
# options that change more than W -> W + scale B A, and the value that leaves them off
_OFF = {"use_dora": False, "fan_in_fan_out": False, "bias": "none", "modules_to_save": None, "rank_pattern": {},
        "alpha_pattern": {}, "lora_bias": False, "layer_replication": None, "alora_invocation_tokens": None}


@dataclass
class Adapter:
    scale: float
    pairs: Dict[str, Tuple[torch.Tensor, torch.Tensor]]  # the changed tensor's name -> (A, B), on the host


def read_adapter(folder: str, spec: ModelSpec) -> Adapter:
    """One `CheckpointError` names everything in the folder that does not fit the model."""
    from ..engine.model import expected_tensors

    path = os.path.join(folder, "adapter_config.json")
    try:
        with open(path) as f:
            cfg = json.load(f)
    except OSError as e:
        raise IoError(f"{path}: cannot open: {e.strerror}") from e
    except ValueError as e:
        raise CheckpointError(f"{path} is not valid JSON: {e}") from None
    if not isinstance(cfg, dict):
        raise CheckpointError(f"{path}: a JSON object is needed")
    r, alpha = cfg.get("r"), cfg.get("lora_alpha")
    if isinstance(r, bool) or not isinstance(r, int) or r < 1:
        raise CheckpointError(f"{path}: r must be a positive integer, got {r!r}")
    if isinstance(alpha, bool) or not isinstance(alpha, (int, float)) or not abs(alpha) < 2.0 ** 127:
        raise CheckpointError(f"{path}: lora_alpha must be a number, got {alpha!r}")
    for key, off in _OFF.items():
        if cfg.get(key, off) not in (off, None, [], {}):
            raise UnsupportedArchitecture(f"{path}: {key} = {cfg[key]!r} is not supported")
    exp = expected_tensors(spec)
    wrong, sides = [], {}
    ckpt = SafetensorsFile(os.path.join(folder, "adapter_model.safetensors"))
    try:
        for key in ckpt.keys():
            side = next((s for s in ("A", "B") if key.endswith(f".lora_{s}.weight")), None)
            name = key[len(PREFIX):-len(".lora_A.weight")] + ".weight" if side else ""
            if not key.startswith(PREFIX) or name not in exp or exp[name][1].role != "matrix":
                wrong.append(f"{key}: no matrix of the model")
                continue
            out, width = exp[name][1].shape
            want = (r, width) if side == "A" else (out, r)
            dtype, shape = ckpt.info(key)
            if tuple(shape) != want or not dtype.is_floating_point:
                wrong.append(f"{key}: expected {list(want)}, found {list(shape)} {dtype}")
                continue
            sides.setdefault(name, {})[side] = ckpt.tensor(key).clone()
    finally:
        ckpt.close()
    wrong += [f"{n}: lora_{'B' if 'A' in s else 'A'} is missing" for n, s in sides.items() if len(s) == 1]
    if wrong or not sides:
        raise CheckpointError(f"{folder} does not fit the '{spec.architecture}' model: "
                              + ("; ".join(wrong) or "no adapter tensors"))
    scale = float(alpha) / (math.sqrt(r) if cfg.get("use_rslora") else r)
    return Adapter(scale, {n: (s["A"], s["B"]) for n, s in sides.items()})
